// Packed batches for sm_100a: the key ranges, query ranges and positions of every token from the batch's document ids, and rotary
// embedding by positions given per token.
#include "common.cuh"
#include "vec8.cuh"
#include "yafsdp_b200.h"

namespace {

// ------------------------------------------------------------------ document mask
// A document is a longest run of equal ids >= 0 in a row of the batch; a negative id is padding.  With start(i), end(i) of token i's
// document, lead(i) = "every token of [start(i), i] is flagged" and run(i) = the end of that leading run:
//   query i sees keys          [start(i), lead(i) ? run(i) : i + 1)        from i - window + 1 on
//   key i is seen by queries   [lead(i) ? start(i) : i, end(i))            before i + window
// so both are single ranges, and both ends of both never decrease along a row, padding's empty [i, i) included.
// A CTA takes 1024 tokens of a row, one per thread.  The tokens at which a document starts, and those that are not flagged, are bits of words
// in shared memory, for the 1024 tokens before and after the tile as well; a token finds the start of its document as the last bit before it and
// the end as the next one behind it.  Only documents longer than that make a CTA read on to the left or the right.  Every CTA works on its
// own: 4 x 32768 tokens 8 us (with one CTA per row, and running maxima over the row, 90 us).  Bound by the latency of the loads and of
// four passes through shared memory.  The CTAs of one long document all read it to its ends, so its time
// grows with the square of its length: 8192 tokens 5.5 us, 131072 49, 2^20 1.7 ms.
constexpr int DM_TILE = 1024, DM_WORDS = DM_TILE / 32;

// Positions around i whose bits are set in 3 x DM_WORDS words that start at position `origin`: the last one <= i, and the first one > i;
// -1 and INT_MAX where there is none.  i is lane's position in word `at`; all lanes of a warp call with the same `at`.
YF_DEVINL int last_at_or_before(const uint32_t* words, int at, int origin) {
  const int lane = threadIdx.x & 31;
  const uint32_t own = words[at] & (0xffffffffu >> (31 - lane));
  // the last word before this one that is not empty: of the 64 words that can be
  const int w1 = at - 1 - lane, w2 = at - 33 - lane;
  const unsigned near = __ballot_sync(0xffffffffu, w1 >= 0 && words[max(w1, 0)] != 0), far = __ballot_sync(0xffffffffu, w2 >= 0 && words[max(w2, 0)] != 0);
  if (own) return origin + at * 32 + 31 - __clz(own);
  if (!(near | far)) return -1;
  const int w = near ? at - __ffs(near) : at - 32 - __ffs(far);
  return origin + w * 32 + 31 - __clz(words[w]);
}
YF_DEVINL int first_behind(const uint32_t* words, int at, int origin) {
  const int lane = threadIdx.x & 31;
  const uint32_t own = lane == 31 ? 0u : words[at] & (0xffffffffu << (lane + 1));
  const int w1 = at + 1 + lane, w2 = at + 33 + lane, n = 3 * DM_WORDS;
  const unsigned near = __ballot_sync(0xffffffffu, w1 < n && words[min(w1, n - 1)] != 0), far = __ballot_sync(0xffffffffu, w2 < n && words[min(w2, n - 1)] != 0);
  if (own) return origin + at * 32 + __ffs(own) - 1;
  if (!(near | far)) return 0x7fffffff;
  const int w = near ? at + __ffs(near) : at + 32 + __ffs(far);
  return origin + w * 32 + __ffs(words[w]) - 1;
}

template <typename ID>
__global__ void __launch_bounds__(DM_TILE) document_mask_kernel(const ID* __restrict__ ids, const uint8_t* __restrict__ prefix,
                                                                int2* __restrict__ spans, int2* __restrict__ key_spans,
                                                                int* __restrict__ positions, int* __restrict__ padding, int S,
                                                                long long ids_stride, long long prefix_stride, int window) {
  __shared__ uint32_t starts[3 * DM_WORDS], plain[3 * DM_WORDS];
  __shared__ int pads[DM_WORDS], found[4];
  const long long row = blockIdx.y;
  const int t0 = blockIdx.x * DM_TILE, origin = t0 - DM_TILE, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ids += row * ids_stride;
  if (prefix) prefix += row * prefix_stride;
  spans += row * S;
  key_spans += row * S;
  positions += row * S;
  padding += row * ((S + 127) / 128);
  // a document starts at p; what is behind the row starts there
  auto starts_at = [&](int p) { return p == 0 || p == S || ids[p] != ids[p - 1]; };
  const int i = t0 + threadIdx.x;
  const bool in = i < S;
  const ID id = in ? ids[i] : (ID)0;
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const int p = origin + part * DM_TILE + threadIdx.x;
    const unsigned s = __ballot_sync(0xffffffffu, p >= 0 && p <= S && starts_at(p));
    const unsigned f = prefix ? __ballot_sync(0xffffffffu, p >= 0 && p < S && prefix[p] == 0) : 0u;
    if (lane == 0) {
      starts[part * DM_WORDS + warp] = s;
      plain[part * DM_WORDS + warp] = f;
    }
  }
  const unsigned dead = __ballot_sync(0xffffffffu, in && id < 0);
  if (lane == 0) pads[warp] = __popc(dead);
  if (threadIdx.x < 4) found[threadIdx.x] = threadIdx.x < 2 ? -1 : 0x7fffffff;
  __syncthreads();
  if (threadIdx.x < DM_TILE / 128 && t0 / 128 + threadIdx.x < (S + 127) / 128) {
    const int* p = pads + 4 * threadIdx.x;
    padding[t0 / 128 + threadIdx.x] = p[0] + p[1] + p[2] + p[3];
  }
  const int at = DM_WORDS + warp;
  int start = last_at_or_before(starts, at, origin), end = first_behind(starts, at, origin);
  int last_plain = -1, next_plain = 0x7fffffff;
  if (prefix) {
    last_plain = last_at_or_before(plain, at, origin);
    next_plain = first_behind(plain, at, origin);
  }
  // A document that is longer than the words reach: on to the left, to the right, until it starts and ends.  (The threads decide together.)
  if (__syncthreads_or(in && start < 0)) {
    for (int p0 = origin; p0 > 0; p0 -= 4 * DM_TILE) {
      int s = -1, f = -1;
#pragma unroll
      for (int k = 1; k <= 4; ++k) {
        const int p = p0 - k * DM_TILE + (int)threadIdx.x;
        if (p < 0) continue;
        if (s < 0 && starts_at(p)) s = p;
        if (f < 0 && prefix && prefix[p] == 0) f = p;
      }
      if (s >= 0) atomicMax(&found[0], s);
      if (f >= 0) atomicMax(&found[1], f);
      if (__syncthreads_or(s >= 0)) break;
    }
    if (start < 0) start = found[0];
    last_plain = max(last_plain, found[1]);
  }
  if (__syncthreads_or(in && end == 0x7fffffff)) {
    for (int p0 = origin + 3 * DM_TILE; p0 <= S; p0 += 4 * DM_TILE) {
      int s = 0x7fffffff, f = 0x7fffffff;
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        const int p = p0 + k * DM_TILE + (int)threadIdx.x;
        if (p > S) continue;
        if (starts_at(p)) s = p;
        if (prefix && p < S && prefix[p] == 0) f = p;
      }
      if (s != 0x7fffffff) atomicMin(&found[2], s);
      if (f != 0x7fffffff) atomicMin(&found[3], f);
      if (__syncthreads_or(s != 0x7fffffff)) break;
    }
    if (end == 0x7fffffff) end = found[2];
    next_plain = min(next_plain, found[3]);
  }
  if (!in) return;
  if (id < 0) {
    spans[i] = key_spans[i] = make_int2(i, i);
    positions[i] = 0;
    return;
  }
  const bool lead = prefix && last_plain < start;
  const int run = min(end, next_plain);
  spans[i] = make_int2(window > 0 ? max(start, i - window + 1) : start, lead ? run : i + 1);
  key_spans[i] = make_int2(lead ? start : i, window > 0 && end - i > window ? i + window : end);
  positions[i] = i - start;
}

// ------------------------------------------------------------------ rotary embedding by positions
// Pair (j, j + half) of a head is turned by positions[axis_j][token] * frequency_j.  The angle is kept as a fraction of a whole turn in
// 64-bit fixed point: table[j] = (2^64 * frequency_j / 2 pi, axis_j), rounded to a whole number, and its product with the position modulo
// 2^64 is exact: off by 2^-65 of a turn for each position (a 32-bit product of position 100000 and frequency 1 is off by up to 0.004 radians).
// The angle's eighth of a turn either side of a whole quarter, to 2^-33 of a turn, is a float and what that conversion left over: the cosine and sine
// of the float are turned by the rest.  (The whole fraction as a float would be off by up to 2^-26.)
// A CTA takes up to RO_TOKENS tokens: every (token, pair) is turned into its cosine and sine once, for all heads of q and k.  A warp takes as many
// heads side by side as its lanes hold vectors of, three times over before it stores anything, so that the memory has enough to do.
// Bound by HBM: every element of q and k is read and written once.  2 x 4096 tokens, 64 / 8 heads of 128 in bf16: 50 to 53 us, 0.88 of the measured copy rate or
// more (67 us with a vector at a time).
constexpr int RO_THREADS = 256, RO_TOKENS = 4, RO_MAX_HALF = 256, RO_BATCH = 3;
struct RotaryArgs {
  const void* src[2];   // q, k
  void* dst[2];
  long long src_token[2], src_head[2], dst_token[2];  // elements between tokens and heads; heads of dst lie side by side
  int heads[2];
  const void* positions;  // [axes][tokens]
  long long axis_stride;  // elements between axes of positions
  const longlong2* table; // [half]
  long long tokens;
  int half;
  int cta_tokens;
  float sign;  // -1: the inverse
};
template <typename T, typename POS>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(RotaryArgs a) {
  // of each eight values the first four, then behind those of all vectors the other four: neighbouring lanes read neighbouring 16 bytes
  __shared__ __align__(16) float cs[RO_TOKENS][RO_MAX_HALF], sn[RO_TOKENS][RO_MAX_HALF];
  const long long t0 = blockIdx.x * (long long)a.cta_tokens;
  const int n = (int)min((long long)a.cta_tokens, a.tokens - t0);
  const POS* pos = reinterpret_cast<const POS*>(a.positions);
  const int half = a.half, vecs = half / 8;
  for (int i = threadIdx.x; i < n * half; i += RO_THREADS) {
    const int t = i / half, j = i - t * half;
    const longlong2 f = __ldg(a.table + j);
    const unsigned long long turn = (unsigned long long)f.x * (unsigned long long)(long long)pos[f.y * a.axis_stride + t0 + t] + (1ull << 31);
    const int hi = (int)(turn >> 32);                           // 2^-32 turns
    const int quarter = (int)(((unsigned)hi + (1u << 29)) >> 30), rest = (int)((unsigned)hi - ((unsigned)quarter << 30));  // rest in [-2^29, 2^29)
    const float near = (float)rest;
    const float d = (float)(rest - (int)near) * 1.4629180792671596e-9f;  // 2^-32 turns in radians: what the float leaves over, up to 16 of them
    float c0, s0;
    sincospif(near * 4.656612873077393e-10f, &s0, &c0);         // 2^-31: half turns in [-1/4, 1/4]
    const float c1 = fmaf(-s0, d, c0), s1 = fmaf(c0, d, s0);
    const float c = quarter & 1 ? s1 : c1, s = quarter & 1 ? c1 : s1;
    const int at = (j & 4 ? half / 2 : 0) + (j >> 3) * 4 + (j & 3);
    cs[t][at] = quarter == 1 || quarter == 2 ? -c : c;
    sn[t][at] = (quarter & 2 ? -s : s) * a.sign;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int abreast = 32 / vecs, hl = lane / vecs, v = lane - hl * vecs;  // heads of a warp, this lane's head and vector
  const int heads = a.heads[0] + a.heads[1], blocks = (heads + abreast - 1) / abreast;
  int t = 0, hb = warp;
  for (int u = warp; u < n * blocks; u += RO_BATCH * (RO_THREADS / 32)) {
    Raw8<T> x[RO_BATCH], y[RO_BATCH];
    T* dst[RO_BATCH];
    int token[RO_BATCH];
#pragma unroll
    for (int k = 0; k < RO_BATCH; ++k, hb += RO_THREADS / 32) {
      while (hb >= blocks) { hb -= blocks; ++t; }
      int h = hb * abreast + hl;
      dst[k] = nullptr;
      token[k] = t;
      if (t < n && hl < abreast && h < heads) {
        const int w = h >= a.heads[0];
        if (w) h -= a.heads[0];
        const T* src = reinterpret_cast<const T*>(a.src[w]) + (t0 + t) * a.src_token[w] + h * a.src_head[w] + v * 8;
        dst[k] = reinterpret_cast<T*>(a.dst[w]) + (t0 + t) * a.dst_token[w] + (long long)h * 2 * half + v * 8;
        x[k] = load_raw8<T>(src);
        y[k] = load_raw8<T>(src + half);
      }
    }
#pragma unroll
    for (int k = 0; k < RO_BATCH; ++k) {
      if (dst[k] == nullptr) continue;
      const float *ct = cs[token[k]], *st = sn[token[k]];
      const float4 c0 = reinterpret_cast<const float4*>(ct)[v], c1 = reinterpret_cast<const float4*>(ct + half / 2)[v];
      const float4 s0 = reinterpret_cast<const float4*>(st)[v], s1 = reinterpret_cast<const float4*>(st + half / 2)[v];
      const F8 c = {{f32x2(c0.x, c0.y), f32x2(c0.z, c0.w), f32x2(c1.x, c1.y), f32x2(c1.z, c1.w)}};
      const F8 s = {{f32x2(s0.x, s0.y), f32x2(s0.z, s0.w), f32x2(s1.x, s1.y), f32x2(s1.z, s1.w)}};
      const F8 m = {{f32x2(-s0.x, -s0.y), f32x2(-s0.z, -s0.w), f32x2(-s1.x, -s1.y), f32x2(-s1.z, -s1.w)}};
      const F8 fx = unpack8<T>(x[k]), fy = unpack8<T>(y[k]);
      store8<T>(dst[k], fma8(fy, m, mul8(fx, c)));
      store8<T>(dst[k] + half, fma8(fx, s, mul8(fy, c)));
    }
  }
}

template <typename T>
int rotary_launch(RotaryArgs a, int pos_64, cudaStream_t st) {
  // few tokens: one each, on as many SMs as there are (45 tokens of 64 heads 2.7 us, 4.3 with four each; 700 of 80 heads 5.4 and 6.7; 2048 12.0
  // either way)
  const long long share = a.tokens / (2 * yf_num_sms());
  a.cta_tokens = share < 1 ? 1 : share > RO_TOKENS ? RO_TOKENS : (int)share;
  const long long ctas = (a.tokens + a.cta_tokens - 1) / a.cta_tokens;
  if (ctas > 0x7fffffffll) return -1;
  if (pos_64) rotary_kernel<T, long long><<<(int)ctas, RO_THREADS, 0, st>>>(a);
  else rotary_kernel<T, int><<<(int)ctas, RO_THREADS, 0, st>>>(a);
  return -(int)cudaGetLastError();
}

}  // namespace

// ids: [B, S] int32 or int64 (ids_64), prefix: [B, S] bytes or null; rows ids_stride / prefix_stride elements apart, tokens side by side.
// spans, key_spans: [B, S, 2] int32; positions: [B, S] int32; padding: [B, ceil(S / 128)] int32, the padded tokens of every 128.
// window: keys at a distance of at least this are hidden (0: none are).
extern "C" int yf_document_mask(const void* ids, int ids_64, const void* prefix, int* spans, int* key_spans, int* positions, int* padding,
                                int B, int S, long long ids_stride, long long prefix_stride, int window, void* stream) {
  if (B <= 0 || B > 65535 || S <= 0 || S > 0x40000000 || window < 0 || !ids || !spans || !key_spans || !positions || !padding) return -1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t* p = reinterpret_cast<const uint8_t*>(prefix);
  int2 *s = reinterpret_cast<int2*>(spans), *k = reinterpret_cast<int2*>(key_spans);
  const dim3 grid((S + DM_TILE - 1) / DM_TILE, B);
  if (ids_64) document_mask_kernel<long long><<<grid, DM_TILE, 0, st>>>(reinterpret_cast<const long long*>(ids), p, s, k, positions, padding, S, ids_stride, prefix_stride, window);
  else document_mask_kernel<int><<<grid, DM_TILE, 0, st>>>(reinterpret_cast<const int*>(ids), p, s, k, positions, padding, S, ids_stride, prefix_stride, window);
  return -(int)cudaGetLastError();
}

// q', k' = q, k turned (sign -1: turned back).  dtype 0 bf16, 1 fp16, 2 fp32; tokens and heads of the inputs are *_token and *_head
// elements apart (multiples of 16 bytes), the outputs' heads lie side by side.  An output may be its input.  head_dim: a multiple of 16,
// at most 512.  positions: [axes][tokens] int32 or int64 (pos_64), axes axis_stride elements apart; table: see rotary_kernel.
extern "C" int yf_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* positions, int pos_64, long long axis_stride,
                         const void* table, long long tokens, int q_heads, int k_heads, int head_dim, long long q_token, long long q_head,
                         long long k_token, long long k_head, long long q_out_token, long long k_out_token, int dtype, int sign, void* stream) {
  const int size = dtype == 2 ? 4 : 2;
  if (tokens <= 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads <= 0 || head_dim <= 0 || head_dim % 16 || head_dim > 2 * RO_MAX_HALF) return -1;
  if (dtype < 0 || dtype > 2 || (sign != 1 && sign != -1) || !positions || !table) return -1;
  if (((q_token | q_head | k_token | k_head | q_out_token | k_out_token) * size) & 15) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out) |
       reinterpret_cast<uintptr_t>(table)) & 15)
    return -1;
  RotaryArgs a;
  a.src[0] = q; a.src[1] = k;
  a.dst[0] = q_out; a.dst[1] = k_out;
  a.src_token[0] = q_token; a.src_token[1] = k_token;
  a.src_head[0] = q_head; a.src_head[1] = k_head;
  a.dst_token[0] = q_out_token; a.dst_token[1] = k_out_token;
  a.heads[0] = q_heads; a.heads[1] = k_heads;
  a.positions = positions;
  a.axis_stride = axis_stride;
  a.table = reinterpret_cast<const longlong2*>(table);
  a.tokens = tokens;
  a.half = head_dim / 2;
  a.sign = (float)sign;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 0) return rotary_launch<__nv_bfloat16>(a, pos_64, st);
  if (dtype == 1) return rotary_launch<__half>(a, pos_64, st);
  return rotary_launch<float>(a, pos_64, st);
}
