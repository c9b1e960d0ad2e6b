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
// One CTA per row: a running maximum from the left finds starts, one of the mirrored row from the right the ends.
constexpr int DM_THREADS = 1024;

YF_DEVINL int warp_scan_max(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}
// inclusive running maximum over the block's threads, on top of `carry` (the same in every thread); returns the block's total in it
YF_DEVINL int block_scan_max(int v, int& carry, int* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan_max(v);
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  const int sums = warp_scan_max(red[lane]);
  const int before = __shfl_sync(0xffffffffu, sums, max(warp, 1) - 1);
  v = max(v, warp == 0 ? carry : max(carry, before));
  carry = max(carry, __shfl_sync(0xffffffffu, sums, 31));
  return v;
}

template <typename ID>
__global__ void __launch_bounds__(DM_THREADS) document_mask_kernel(const ID* __restrict__ ids, const uint8_t* __restrict__ prefix,
                                                                   int2* __restrict__ spans, int2* __restrict__ key_spans,
                                                                   int* __restrict__ positions, int* __restrict__ padding, int S,
                                                                   long long ids_stride, long long prefix_stride, int window) {
  __shared__ int red[32], pads[32];
  const long long row = blockIdx.x;
  ids += row * ids_stride;
  if (prefix) prefix += row * prefix_stride;
  spans += row * S;
  key_spans += row * S;
  positions += row * S;
  padding += row * ((S + 127) / 128);
  const int chunks = (S + DM_THREADS - 1) / DM_THREADS;
  // left to right: start(i), lead(i) (parked in key_spans by the thread that fetches them below)
  int last_start = 0, last_plain = -1;
  for (int c = 0; c < chunks; ++c) {
    const int i = c * DM_THREADS + threadIdx.x;
    const bool in = i < S;
    const ID id = in ? ids[i] : (ID)-1;
    const bool starts = in && (i == 0 || ids[i - 1] != id);
    const int start = block_scan_max(starts ? i : 0, last_start, red);
    int lead = 0;
    if (prefix) {
      const bool plain = in && prefix[i] == 0;
      lead = block_scan_max(plain ? i : -1, last_plain, red) < start;
    }
    if (in) key_spans[i] = make_int2(start, lead);
    const unsigned dead = __ballot_sync(0xffffffffu, in && id < 0);
    if ((threadIdx.x & 31) == 0) pads[threadIdx.x >> 5] = __popc(dead);
    __syncthreads();
    if (threadIdx.x < 8 && c * 8 + threadIdx.x < (S + 127) / 128)
      padding[c * 8 + threadIdx.x] = pads[4 * threadIdx.x] + pads[4 * threadIdx.x + 1] + pads[4 * threadIdx.x + 2] + pads[4 * threadIdx.x + 3];
  }
  // right to left: end(i), run(i), as running maxima of the negated positions
  int next_end = -S, next_plain = -S;
  for (int c = chunks - 1; c >= 0; --c) {
    const int i = c * DM_THREADS + (DM_THREADS - 1 - (int)threadIdx.x);
    const bool in = i < S;
    const ID id = in ? ids[i] : (ID)-1;
    const bool ends = in && (i == S - 1 || ids[i + 1] != id);
    const int end = -block_scan_max(ends ? -(i + 1) : -S, next_end, red);
    int run = end;
    if (prefix) run = min(run, -block_scan_max(in && prefix[i] == 0 ? -i : -S, next_plain, red));
    if (!in) continue;
    if (id < 0) {
      spans[i] = key_spans[i] = make_int2(i, i);
      positions[i] = 0;
      continue;
    }
    const int2 parked = key_spans[i];
    const int start = parked.x;
    const bool lead = parked.y != 0;
    const int far = window > 0 && end - i > window ? i + window : end;
    spans[i] = make_int2(window > 0 ? max(start, i - window + 1) : start, lead ? run : i + 1);
    key_spans[i] = make_int2(lead ? start : i, far);
    positions[i] = i - start;
  }
}

// ------------------------------------------------------------------ rotary embedding by positions
// Pair (j, j + half) of a head is turned by positions[axis_j][token] * frequency_j.  The angle is kept as a fraction of a whole turn in
// 64-bit fixed point: table[j] = (2^64 * frequency_j / 2 pi, axis_j), and the product with the integer position modulo 2^64 is exact, so
// far positions lose nothing (a 32-bit product of position 100000 and frequency 1 is off by up to 0.004).
// A CTA takes RO_TOKENS tokens: every (token, pair) is turned into its cosine and sine once, for all heads of q and k.
// Bound by HBM: every element of q and k is read and written once.
constexpr int RO_THREADS = 256, RO_TOKENS = 4, RO_MAX_HALF = 256;
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
  float sign;  // -1: the inverse
};
template <typename T, typename POS>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(RotaryArgs a) {
  __shared__ float cs[RO_TOKENS][RO_MAX_HALF], sn[RO_TOKENS][RO_MAX_HALF];
  const long long t0 = blockIdx.x * (long long)RO_TOKENS;
  const int n = (int)min((long long)RO_TOKENS, a.tokens - t0);
  const POS* pos = reinterpret_cast<const POS*>(a.positions);
  for (int i = threadIdx.x; i < n * a.half; i += RO_THREADS) {
    const int t = i / a.half, j = i - t * a.half;
    const longlong2 f = __ldg(a.table + j);
    const unsigned long long turn = (unsigned long long)f.x * (unsigned long long)(long long)pos[f.y * a.axis_stride + t0 + t];
    float c, s;
    sincospif((float)(int)(turn >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: half turns in [-1, 1]
    cs[t][j] = c;
    sn[t][j] = s * a.sign;
  }
  __syncthreads();
  const int vecs = a.half / 8, per_token = (a.heads[0] + a.heads[1]) * vecs;
  for (int i = threadIdx.x; i < n * per_token; i += RO_THREADS) {
    const int t = i / per_token, r = i - t * per_token;
    int h = r / vecs;
    const int v = (r - h * vecs) * 8;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    const T* src = reinterpret_cast<const T*>(a.src[w]) + (t0 + t) * a.src_token[w] + h * a.src_head[w] + v;
    T* dst = reinterpret_cast<T*>(a.dst[w]) + (t0 + t) * a.dst_token[w] + (long long)h * 2 * a.half + v;
    float x[8], y[8], ox[8], oy[8];
    load_f8<T>(src, x);
    load_f8<T>(src + a.half, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = cs[t][v + j], s = sn[t][v + j];
      ox[j] = x[j] * c - y[j] * s;
      oy[j] = y[j] * c + x[j] * s;
    }
    store_f8<T>(dst, ox);
    store_f8<T>(dst + a.half, oy);
  }
}

template <typename T>
int rotary_launch(const RotaryArgs& a, int pos_64, cudaStream_t st) {
  const long long ctas = (a.tokens + RO_TOKENS - 1) / RO_TOKENS;
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
  if (B <= 0 || S <= 0 || S > 0x40000000 || window < 0 || !ids || !spans || !key_spans || !positions || !padding) return -1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t* p = reinterpret_cast<const uint8_t*>(prefix);
  int2 *s = reinterpret_cast<int2*>(spans), *k = reinterpret_cast<int2*>(key_spans);
  if (ids_64) document_mask_kernel<long long><<<B, DM_THREADS, 0, st>>>(reinterpret_cast<const long long*>(ids), p, s, k, positions, padding, S, ids_stride, prefix_stride, window);
  else document_mask_kernel<int><<<B, DM_THREADS, 0, st>>>(reinterpret_cast<const int*>(ids), p, s, k, positions, padding, S, ids_stride, prefix_stride, window);
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
