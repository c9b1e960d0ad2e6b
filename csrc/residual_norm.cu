// The residual step between two blocks of a decoder for sm_100a:
//   u = y * rsqrt(mean(y^2) + eps) * post      (the norm after the block; u = y without one)
//   h = x + scale * gate * u                    (gate: none, one row for a group of tokens, or a row per token)
//   n = h * rsqrt(mean(h^2) + eps) * weight     (the norm before the next block)
// and its gradients.  With dh, dn the gradients of h and n, and hats for what a norm has divided:
//   g = dh + r_h (dn weight - hhat mean(dn weight hhat)) = dx
//   e = scale gate g,  dy = r_y (e post - yhat mean(e post yhat)),
//   dweight = sum dn hhat,  dpost = sum e yhat,  dgate = scale sum g u  over the tokens that share the row.
// Bound by HBM: forward reads x, y and writes h, n once; backward reads x, y, dh, dn and writes dx, dy once.  h is formed anew in
// the backward pass: the rounded h would take as many bytes and lose bits.  All sums are fp32, and in a fixed order but for
// the squares of the weights' gradients, which the parameter kernel's blocks add to their target by atomics.
// 8192 x 8192 in bf16: 107 us forward, 159 backward, 5.0 TB/s of 6.5 for a copy (133 and 204 with plain loads): a row's two reductions stand behind each
// other.  Blocks of 512 threads forward take as long, three blocks per SM spill (120), 320 threads for rows of 5120 gain nothing.
// Further from a copy's rate: backward above width 4096 with fewer rows or a width between the classes (one block of 512 threads per SM waits at both
// reductions; 4096 x 5120 53 to 75 us by gate and post norm, 2048 x 8192 39 to 54: at most 5.1 TB/s); width 512 (8192 rows 7 to 8 us forward and 16
// to 26 backward, with everything in the L2: a warp has 2 to 4 rows, so starts and ends count); and fp32, whose backward kernels spill 32 to 436
// bytes a thread (4096 x 4096 80 us; bf16 and fp16 up to 132 with a gate per token at widths to 2048).
#include "common.cuh"
#include "vec8.cuh"
#include "yafsdp_b200.h"

YF_TU_STATUS()

namespace {

// TPR threads take a row at a time (16 elements each, 32 in the forward pass of wide rows: two blocks of 256 threads overlap their reductions better
// than one of 512), a block of at least 256 threads as many rows as that makes.  Every row group has a ring of shared memory into
// which bulk copies bring its next rows while it works on one, so that the memory is busy during the two reductions of a row, and the
// registers hold one row only.
template <int TPR>
constexpr int BLOCK = TPR < 256 ? 256 : TPR;
template <int TPR, int NV>
constexpr int FWD_BLOCKS = NV == 2 ? 3 : 2;  // per SM
template <int TPR>
constexpr int BWD_BLOCKS = TPR < 512 ? 2 : 1;
constexpr int MAX_STAGES = 4;
// Rows are counted in 32 bits; up to here a walker's next rows still are, which lie up to 4 x 2368 behind its own.
constexpr int MAX_ROWS = 0x7fffffff - (1 << 20);
// What the rings of an SM's blocks take together: 160 KB, which leaves room for the L1 that the weights come from, and more only for rows of which
// not even one would fit.
constexpr int RING_BYTES = 160 * 1024, RING_BYTES_MOST = 192 * 1024;
int ring_stages(int stage_bytes, int blocks) {
  const int n = RING_BYTES / blocks / stage_bytes;
  return n < 1 ? 1 : n > MAX_STAGES ? MAX_STAGES : n;
}

YF_DEVINL bool group_bar_or(int tpr, int group, bool flag) {
  // literal barrier numbers: a computed one reserves all sixteen
  if (group == 0) return named_bar_or(1, tpr, flag);
  if (group == 1) return named_bar_or(2, tpr, flag);
  if (group == 2) return named_bar_or(3, tpr, flag);
  return named_bar_or(4, tpr, flag);
}
// sum over the TPR threads of a row; false when one of them says so.  What they read before it is read behind it.  `slots`: one float per warp of
// the block, not used again before the row's threads have met at another barrier.
template <int TPR>
YF_DEVINL bool row_sum(float& v, float* slots, int group, bool ok = true) {
  v = warp_sum(v);
  if (TPR == 32) {
    ok = __all_sync(0xffffffffu, ok);
    __syncwarp();  // the vote does not order memory: what the lanes have read of a stage comes before the copy into it
    return ok;
  }
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  if (group_bar_or(TPR, group, !ok)) return false;
  v = 0.f;
#pragma unroll
  for (int g = 0; g < TPR / 32; ++g) v += slots[group * (TPR / 32) + g];
  return true;
}

struct NormArgs {
  const void *x, *y, *weight, *post, *gate;  // post, gate: may be null
  void *h, *n;
  float* rstd;  // [T, 2]: r_y (with post), r_h; may be null
  const void *dh, *dn;  // one of them may be null: zeros
  void *dx, *dy, *dgate;
  float *w_parts, *z_parts;  // [CTAs, D]: sums of dn hhat and of g yhat (g y without post; gate g yhat with a gate per token)
  float scale, eps;
  int T, D;
  int group_rows;    // tokens that share a row of the gate
  int ctas_per_group;
  int token_gate;    // a row of the gate for every token
  int stages;
};

// The ring of a row group: `tensors` rows of D elements side by side in each stage.
template <typename T, int TPR>
struct Ring {
  uint8_t* base;
  uint64_t* full;
  const void* src[5];
  int tensors, row_bytes, stages;
  int stage, phase;

  YF_DEVINL void start(uint8_t* smem, uint64_t* bars, int group, int n_stages, int n_tensors, int D) {
    tensors = n_tensors;
    row_bytes = D * (int)sizeof(T);
    stages = n_stages;
    base = smem + (size_t)group * stages * tensors * row_bytes;
    full = bars + group * MAX_STAGES;
    stage = phase = 0;
  }
  // one thread: row `row` of every tensor into stage s
  YF_DEVINL void fetch(int s, long long row) {
    mbar_expect_tx(&full[s], (uint32_t)(tensors * row_bytes));
#pragma unroll
    for (int t = 0; t < 5; ++t)
      if (t < tensors)
        bulk_load(base + (size_t)(s * tensors + t) * row_bytes, reinterpret_cast<const uint8_t*>(src[t]) + row * row_bytes, (uint32_t)row_bytes, &full[s]);
  }
  YF_DEVINL const T* row(int t) const { return reinterpret_cast<const T*>(base + (size_t)(stage * tensors + t) * row_bytes); }
  YF_DEVINL bool wait(int site) { return mbar_wait(&full[stage], phase, site); }
  YF_DEVINL void next() {
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
};

// scale * gate * post of the thread's columns: what a normalised y is multiplied by, and one vector for what would be two
template <typename T, int NV, int TPR>
YF_DEVINL void factors(F8 (&f)[NV], float scale, const void* gate, const void* post, int tr, int nvec) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tr + TPR * i;
    f[i] = splat8(scale);
    if (v < nvec) {
      if (gate) f[i] = mul8(f[i], unpack8<T>(load_raw8<T>(reinterpret_cast<const T*>(gate) + v * 8)));
      if (post) f[i] = mul8(f[i], unpack8<T>(load_raw8<T>(reinterpret_cast<const T*>(post) + v * 8)));
    }
  }
}

// A row group walks over adjacent rows, so that the gate's row seldom changes.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(BLOCK<TPR>, FWD_BLOCKS<TPR, NV>) residual_norm_fwd_kernel(NormArgs a) {
  constexpr int ROWS = BLOCK<TPR> / TPR;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[ROWS * MAX_STAGES];
  __shared__ float slots[2][2][BLOCK<TPR> / 32];
  const int group = threadIdx.x / TPR, tr = threadIdx.x % TPR;
  const int nvec = a.D / 8;
  const int walkers = gridDim.x * ROWS, each = (a.T + walkers - 1) / walkers;
  const int first = min((long long)(blockIdx.x * ROWS + group) * each, (long long)a.T), end = min((long long)first + each, (long long)a.T);
  Ring<T, TPR> ring;
  ring.start(smem, bars, group, a.stages, a.token_gate ? 3 : 2, a.D);
  ring.src[0] = a.x;
  ring.src[1] = a.y;
  ring.src[2] = a.gate;
  if (threadIdx.x == 0) {
    for (int i = 0; i < ROWS * MAX_STAGES; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  if (tr == 0)
    for (int s = 0; s < a.stages; ++s)
      if (first + s < end) ring.fetch(s, first + s);
  const T *w = reinterpret_cast<const T*>(a.weight), *gate = reinterpret_cast<const T*>(a.gate);
  int in_group = 0;  // rows until the gate's row changes
  if (gate && !a.token_gate && first < end) {
    gate += (long long)(first / a.group_rows) * a.D;
    in_group = a.group_rows - first % a.group_rows;
  }
  F8 f[NV];
  factors<T, NV, TPR>(f, a.scale, a.token_gate ? nullptr : gate, a.post, tr, nvec);
  int parity = 0;
  for (int row = first; row < end; ++row, parity ^= 1) {
    const long long at = (long long)row * a.D;
    // a wait that runs out ends the work of the row's threads together
    const bool ok = ring.wait(600);
    const T *x = ring.row(0), *y = ring.row(1);
    F8 h[NV], u[NV];
    uint64_t ss = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        h[i] = unpack8<T>(load_raw8<T>(x + v * 8));
        u[i] = unpack8<T>(load_raw8<T>(y + v * 8));
        dot8(ss, u[i], u[i]);
        if (a.token_gate) u[i] = mul8(u[i], unpack8<T>(load_raw8<T>(ring.row(2) + v * 8)));
      }
    }
    // behind this sum the row is in registers, and its stage is free
    float sum = both(ss);
    if (!row_sum<TPR>(sum, slots[0][parity], group, ok)) break;
    if (tr == 0 && row + a.stages < end) ring.fetch(ring.stage, row + a.stages);
    ring.next();
    const float ry = a.post ? rsqrtf(sum / (float)a.D + a.eps) : 1.f;
    ss = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        h[i] = fma8(mul8(u[i], ry), f[i], h[i]);
        dot8(ss, h[i], h[i]);
        store8<T>(reinterpret_cast<T*>(a.h) + at + v * 8, h[i]);
      }
    }
    sum = both(ss);
    row_sum<TPR>(sum, slots[1][parity], group);
    const float rh = rsqrtf(sum / (float)a.D + a.eps);
    if (tr == 0 && a.rstd) reinterpret_cast<float2*>(a.rstd)[row] = make_float2(ry, rh);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) store8<T>(reinterpret_cast<T*>(a.n) + at + v * 8, mul8(mul8(h[i], rh), unpack8<T>(load_raw8<T>(w + v * 8))));
    }
    if (in_group > 0 && --in_group == 0 && row + 1 < end) {
      gate += a.D;
      in_group = a.group_rows;
      factors<T, NV, TPR>(f, a.scale, gate, a.post, tr, nvec);
    }
  }
}

// A CTA walks over the rows of one group of tokens (all tokens where the gate is per token); its threads hold the same columns of every
// row and sum the parameters' gradients in registers on the way.
template <typename T, int TPR, bool TOKEN_GATE>
__global__ void __launch_bounds__(BLOCK<TPR>, BWD_BLOCKS<TPR>) residual_norm_bwd_kernel(NormArgs a) {
  constexpr int THREADS = BLOCK<TPR>, ROWS = THREADS / TPR, NV = 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[ROWS * MAX_STAGES];
  __shared__ float slots[2][2][THREADS / 32];
  const int group = threadIdx.x / TPR, tr = threadIdx.x % TPR;
  const int nvec = a.D / 8;
  const int part = blockIdx.x % a.ctas_per_group, gg = blockIdx.x / a.ctas_per_group;
  const int rows = TOKEN_GATE ? a.T : a.group_rows;
  const int first = part * ROWS + group, step = a.ctas_per_group * ROWS;
  const long long row0 = (long long)gg * rows;
  const float inv_d = 1.f / (float)a.D;
  const T* w = reinterpret_cast<const T*>(a.weight);
  Ring<T, TPR> ring;
  ring.src[0] = a.x;
  ring.src[1] = a.y;
  // the gradients that there are, then the gate
  const int at_dn = a.dh ? 3 : 2, at_gate = at_dn + (a.dn ? 1 : 0);
  ring.src[2] = a.dh ? a.dh : a.dn ? a.dn : a.gate;
  ring.src[3] = a.dh && a.dn ? a.dn : a.gate;
  ring.src[4] = a.gate;
  ring.start(smem, bars, group, a.stages, at_gate + (TOKEN_GATE ? 1 : 0), a.D);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ROWS * MAX_STAGES; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  if (tr == 0)
    for (int s = 0; s < a.stages; ++s)
      if (first + s * step < rows) ring.fetch(s, row0 + first + s * step);
  F8 acc_w[NV], acc_z[NV], f[NV];  // f: without the gate where it is per token
#pragma unroll
  for (int i = 0; i < NV; ++i) acc_w[i] = acc_z[i] = splat8(0.f);
  factors<T, NV, TPR>(f, a.scale, TOKEN_GATE || !a.gate ? nullptr : reinterpret_cast<const T*>(a.gate) + (long long)gg * a.D, a.post, tr, nvec);
  int parity = 0;
  const float2* rstd = reinterpret_cast<const float2*>(a.rstd) + row0;
  float2 rs = first < rows ? rstd[first] : make_float2(0.f, 0.f);  // read a row ahead
  for (int r = first; r < rows; r += step, parity ^= 1) {
    const long long row = row0 + r, at = row * a.D;
    const float ry = rs.x, rh = rs.y;
    if (r + step < rows) rs = rstd[r + step];
    const bool ok = ring.wait(601);
    Raw8<T> yr[NV], dhr[NV], gr[NV];
    F8 hv[NV], cv[NV];
    uint64_t dot = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        yr[i] = load_raw8<T>(ring.row(1) + v * 8);
        if (a.dh) dhr[i] = load_raw8<T>(ring.row(2) + v * 8);
        if (TOKEN_GATE) gr[i] = load_raw8<T>(ring.row(at_gate) + v * 8);
        F8 u = mul8(unpack8<T>(yr[i]), ry);
        if (TOKEN_GATE) u = mul8(u, unpack8<T>(gr[i]));
        hv[i] = mul8(fma8(u, f[i], unpack8<T>(load_raw8<T>(ring.row(0) + v * 8))), rh);  // hhat
        cv[i] = splat8(0.f);
        if (a.dn) {
          const F8 dn = unpack8<T>(load_raw8<T>(ring.row(at_dn) + v * 8));
          acc_w[i] = fma8(dn, hv[i], acc_w[i]);
          cv[i] = mul8(dn, unpack8<T>(load_raw8<T>(w + v * 8)));
          dot8(dot, cv[i], hv[i]);
        }
      }
    }
    // behind this sum the row is in registers, and its stage is free
    float sum = both(dot);
    if (!row_sum<TPR>(sum, slots[0][parity], group, ok)) break;
    if (tr == 0 && r + (long long)a.stages * step < rows) ring.fetch(ring.stage, row + (long long)a.stages * step);
    ring.next();
    sum *= -inv_d;
    dot = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        F8 g = fma8(hv[i], sum, cv[i]);
        g = a.dh ? fma8(g, rh, unpack8<T>(dhr[i])) : mul8(g, rh);
        store8<T>(reinterpret_cast<T*>(a.dx) + at + v * 8, g);
        hv[i] = mul8(unpack8<T>(yr[i]), ry);  // yhat (y itself without post)
        if (TOKEN_GATE) {
          const F8 gy = mul8(g, hv[i]), gate = unpack8<T>(gr[i]);
          store8<T>(reinterpret_cast<T*>(a.dgate) + at + v * 8, mul8(gy, f[i]));
          acc_z[i] = fma8(gy, gate, acc_z[i]);
          g = mul8(g, gate);
        } else {
          acc_z[i] = fma8(g, hv[i], acc_z[i]);
        }
        cv[i] = mul8(g, f[i]);  // e post
        dot8(dot, cv[i], hv[i]);
      }
    }
    sum = both(dot);
    if (a.post) row_sum<TPR>(sum, slots[1][parity], group);
    sum = a.post ? -sum * inv_d : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) store8<T>(reinterpret_cast<T*>(a.dy) + at + v * 8, mul8(fma8(hv[i], sum, cv[i]), ry));
    }
  }
  float* sums = reinterpret_cast<float*>(smem);  // ROWS > 1: every row has been read by now
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* parts = k == 0 ? a.w_parts : a.z_parts;
    if (parts == nullptr) continue;
    float acc[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = f32x2_split(k == 0 ? acc_w[i].p[j] : acc_z[i].p[j]);
        acc[i][2 * j] = t.x;
        acc[i][2 * j + 1] = t.y;
      }
    if (ROWS > 1) {  // the row groups in turn: the last one ends up with the sum
      __syncthreads();
#pragma unroll 1
      for (int o = 0; o < ROWS; ++o) {
        if (group == o) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            float* at = sums + (tr + TPR * i) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (o > 0) acc[i][j] += at[j];
              at[j] = acc[i][j];
            }
          }
        }
        __syncthreads();
      }
    }
    if (group == ROWS - 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = tr + TPR * i;
        if (v < nvec) {
          float4* at = reinterpret_cast<float4*>(parts + (long long)blockIdx.x * a.D + v * 8);
          at[0] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
          at[1] = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
        }
      }
    }
  }
}

struct ParamArgs {
  const float *w_parts, *z_parts;  // z_parts may be null
  const void *post, *gate;
  void *dw, *dpost, *dgate;        // dpost, dgate may be null
  int dw_kind, dpost_kind;         // 0: the type of the activations, 1: fp32, 2: fp32, added to what is there
  float *dw_sumsq, *dpost_sumsq;   // optional, += the squares of what was written
  float scale;
  int D, groups, ctas_per_group, token_gate;
};
template <typename T>
YF_DEVINL float store_param(void* dst, int kind, int col, float v) {
  if (kind == 0) {
    if (sizeof(T) == 4) reinterpret_cast<float*>(dst)[col] = v;
    else reinterpret_cast<T*>(dst)[col] = (T)v;
  } else {
    float* at = reinterpret_cast<float*>(dst) + col;
    if (kind == 2) v += *at;
    *at = v;
  }
  return v;
}
// The parameters' gradients from the CTAs' sums: 32 columns per CTA, 32 threads per column; every sum in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_param_kernel(ParamArgs a) {
  __shared__ float part[32][33];
  const int c = threadIdx.x & 31, lane_row = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c, mine = blockIdx.x * 32 + lane_row;  // reads column `col`, finishes column `mine`
  const int n = a.groups * a.ctas_per_group;
  auto finish = [&](float s) {  // the sum over lane_row of column `mine`, in every lane of the warp
    __syncthreads();
    part[lane_row][c] = s;
    __syncthreads();
    return warp_sum(part[c][lane_row]);
  };
  auto norm = [&](float* target, float v) {  // *target += the squares of this CTA's columns
    if (target == nullptr) return;
    __syncthreads();
    if (c == 0) part[0][lane_row] = mine < a.D ? v * v : 0.f;
    __syncthreads();
    if (lane_row == 0) {
      const float total = warp_sum(part[0][c]);
      if (c == 0) atomicAdd(target, total);
    }
  };
  float s = 0.f;
  if (col < a.D)
    for (int i = lane_row; i < n; i += 32) s += a.w_parts[(long long)i * a.D + col];
  s = finish(s);
  if (c == 0 && mine < a.D) s = store_param<T>(a.dw, a.dw_kind, mine, s);
  norm(a.dw_sumsq, s);
  if (a.z_parts == nullptr) return;
  const T *gate = reinterpret_cast<const T*>(a.gate), *post = reinterpret_cast<const T*>(a.post);
  float dpost = 0.f;
  if (a.token_gate) {
    if (col < a.D)
      for (int i = lane_row; i < n; i += 32) dpost += a.z_parts[(long long)i * a.D + col];
    dpost = a.scale * finish(dpost);
  } else if (a.ctas_per_group == 1) {  // a thread has whole groups
    if (col < a.D) {
      const float p = post ? (float)post[col] : 1.f;
      for (int i = lane_row; i < n; i += 32) {
        const long long at = (long long)i * a.D + col;
        const float z = a.scale * a.z_parts[at];
        dpost += z * (gate ? (float)gate[at] : 1.f);
        if (a.dgate) reinterpret_cast<T*>(a.dgate)[at] = (T)(z * p);
      }
    }
    dpost = finish(dpost);
  } else {
    for (int g = 0; g < a.groups; ++g) {
      float z = 0.f;
      if (col < a.D)
        for (int i = lane_row; i < a.ctas_per_group; i += 32) z += a.z_parts[((long long)g * a.ctas_per_group + i) * a.D + col];
      z = a.scale * finish(z);
      if (mine < a.D) {
        const long long at = (long long)g * a.D + mine;
        dpost += z * (gate ? (float)gate[at] : 1.f);
        if (a.dgate && c == 0) reinterpret_cast<T*>(a.dgate)[at] = (T)(z * (post ? (float)post[mine] : 1.f));
      }
    }
  }
  if (a.dpost == nullptr) return;
  if (c == 0 && mine < a.D) dpost = store_param<T>(a.dpost, a.dpost_kind, mine, dpost);
  norm(a.dpost_sumsq, dpost);
}

int row_threads(int D) {  // threads that hold a row: 16 elements each
  int t = 32;
  while (t * 16 < D) t *= 2;
  return t;
}
int rows_per_block(int D) { return row_threads(D) < 256 ? 256 / row_threads(D) : 1; }
// CTAs that walk over one group of tokens: what is resident altogether, no more than there are rows for
int ctas_per_group(int T, int D, int groups) {
  const int rows = rows_per_block(D), in_group = T / groups;
  int want = (row_threads(D) < 512 ? BWD_BLOCKS<256> : BWD_BLOCKS<512>) * yf_num_sms() / groups;
  const int most = (in_group + rows - 1) / rows;
  if (want > most) want = most;
  return want < 1 ? 1 : want;
}

// sums: bytes that the sums of the row groups want
int launch_rows(void (*kernel)(NormArgs), bool (&optin)[64], NormArgs a, int stage_bytes, int blocks, int sums, int grid, int threads, cudaStream_t st) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (!optin[dev]) {  // the shared-memory opt-in is a per-device attribute
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES_MOST);
    if (e != cudaSuccess) return -(int)e;
    optin[dev] = true;
  }
  if (int rc = yf_tu_bind_status()) return rc;
  a.stages = ring_stages(stage_bytes, blocks);
  const int bytes = a.stages * stage_bytes;
  if (bytes > RING_BYTES_MOST) return -1;
  kernel<<<grid, threads, bytes < sums ? sums : bytes, st>>>(a);
  return -(int)cudaGetLastError();
}
template <typename T, int N, int NV>
int fwd_launch_n(const NormArgs& a, cudaStream_t st) {
  static bool optin[64] = {};
  constexpr int rows = BLOCK<N> / N;
  int grid = (a.T + rows - 1) / rows;
  const int most = FWD_BLOCKS<N, NV> * yf_num_sms();
  if (grid > most) grid = most;
  return launch_rows(residual_norm_fwd_kernel<T, N, NV>, optin, a, (a.token_gate ? 3 : 2) * rows * a.D * (int)sizeof(T), FWD_BLOCKS<N, NV>, 0, grid, BLOCK<N>, st);
}
template <typename T, int N>
int bwd_launch_n(const NormArgs& a, int grid, cudaStream_t st) {
  static bool optin[2][64] = {};
  const int tensors = 2 + (a.dh ? 1 : 0) + (a.dn ? 1 : 0) + (a.token_gate ? 1 : 0), stage = tensors * (BLOCK<N> / N) * a.D * (int)sizeof(T);
  return a.token_gate ? launch_rows(residual_norm_bwd_kernel<T, N, true>, optin[1], a, stage, BWD_BLOCKS<N>, N * 64, grid, BLOCK<N>, st)
                      : launch_rows(residual_norm_bwd_kernel<T, N, false>, optin[0], a, stage, BWD_BLOCKS<N>, N * 64, grid, BLOCK<N>, st);
}
template <typename T>
int fwd_launch(const NormArgs& a, cudaStream_t st) {
  switch (row_threads(a.D)) {
    case 32: return fwd_launch_n<T, 32, 2>(a, st);
    case 64: return fwd_launch_n<T, 64, 2>(a, st);
    case 128: return fwd_launch_n<T, 128, 2>(a, st);
    case 256: return fwd_launch_n<T, 256, 2>(a, st);
    default: return fwd_launch_n<T, 256, 4>(a, st);
  }
}
template <typename T>
int bwd_launch(const NormArgs& a, const ParamArgs& p, cudaStream_t st) {
  const int grid = p.groups * p.ctas_per_group;
  int rc = 0;
  switch (row_threads(a.D)) {
    case 32: rc = bwd_launch_n<T, 32>(a, grid, st); break;
    case 64: rc = bwd_launch_n<T, 64>(a, grid, st); break;
    case 128: rc = bwd_launch_n<T, 128>(a, grid, st); break;
    case 256: rc = bwd_launch_n<T, 256>(a, grid, st); break;
    default: rc = bwd_launch_n<T, 512>(a, grid, st); break;
  }
  if (rc) return rc;
  residual_norm_param_kernel<T><<<(a.D + 31) / 32, 1024, 0, st>>>(p);
  return -(int)cudaGetLastError();
}

bool misaligned(const void* const* p, int n) {
  uintptr_t bits = 0;
  for (int i = 0; i < n; ++i) bits |= reinterpret_cast<uintptr_t>(p[i]);
  return (bits & 15) != 0;
}
bool bad_shape(int T, int D, int gate_rows, const void* gate, int dtype) {
  if (T <= 0 || T > MAX_ROWS || D <= 0 || D % 8 || D > 8192 || dtype < 0 || dtype > 2) return true;
  return gate != nullptr ? gate_rows <= 0 || T % gate_rows != 0 : gate_rows != 0;
}

}  // namespace

// x, y, h, n: [T, D] without gaps; weight, post: [D]; gate: [gate_rows, D], row t / (T / gate_rows) for token t (gate_rows 0 without one); all
// of one type (dtype 0 bf16, 1 fp16, 2 fp32), 16-byte aligned, D a multiple of 8 up to 8192, T up to 2^31 - 2^20 - 1.  rstd: [T, 2] fp32 for the backward
// pass, or null.
extern "C" int yf_residual_norm_fwd(const void* x, const void* y, const void* weight, const void* post, const void* gate, int gate_rows, void* h,
                                    void* n, float* rstd, int T, int D, float scale, float eps, int dtype, void* stream) {
  const void* ptrs[] = {x, y, weight, post, gate, h, n, rstd};
  if (bad_shape(T, D, gate_rows, gate, dtype) || !x || !y || !weight || !h || !n || misaligned(ptrs, 8)) return -1;
  NormArgs a = {};
  a.x = x; a.y = y; a.weight = weight; a.post = post; a.gate = gate;
  a.h = h; a.n = n;
  a.rstd = rstd;
  a.T = T; a.D = D;
  a.scale = scale; a.eps = eps;
  a.group_rows = gate ? T / gate_rows : T;
  a.token_gate = gate != nullptr && gate_rows == T;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == 0 ? fwd_launch<__nv_bfloat16>(a, st) : dtype == 1 ? fwd_launch<__half>(a, st) : fwd_launch<float>(a, st);
}

// Rows of [rows, D] fp32 scratch that the backward pass wants (twice that with a post norm or a gate).
extern "C" int yf_residual_norm_parts(int T, int D, int gate_rows) {
  if (T <= 0 || T > MAX_ROWS || D <= 0 || D % 8 || D > 8192 || gate_rows < 0 || (gate_rows > 0 && T % gate_rows)) return -1;
  const int groups = gate_rows == 0 || gate_rows == T ? 1 : gate_rows;
  const long long n = (long long)groups * ctas_per_group(T, D, groups);
  return n > 0x7fffffff ? -1 : (int)n;
}

// Gradients of yf_residual_norm_fwd.  dh, dn: one of them may be null (zeros).  parts: yf_residual_norm_parts rows of D floats, twice as many with
// post or gate; parts_floats says how many there are.  dw, dpost: kind 0 the type of the activations, 1 fp32, 2 fp32 that is added to;
// *_sumsq (optional): += the squares of what was written.
extern "C" int yf_residual_norm_bwd(const void* x, const void* y, const void* weight, const void* post, const void* gate, int gate_rows,
                                    const float* rstd, const void* dh, const void* dn, void* dx, void* dy, void* dw, int dw_kind, float* dw_sumsq,
                                    void* dpost, int dpost_kind, float* dpost_sumsq, void* dgate, float* parts, long long parts_floats, int T, int D,
                                    float scale, int dtype, void* stream) {
  const void* ptrs[] = {x, y, weight, post, gate, rstd, dh, dn, dx, dy, dgate, parts};
  if (bad_shape(T, D, gate_rows, gate, dtype) || !x || !y || !weight || !rstd || !dx || !dy || !dw || !parts || misaligned(ptrs, 12)) return -1;
  if ((!dh && !dn) || (post != nullptr) != (dpost != nullptr) || (gate != nullptr) != (dgate != nullptr)) return -1;
  if (dw_kind < 0 || dw_kind > 2 || dpost_kind < 0 || dpost_kind > 2) return -1;
  const bool token_gate = gate != nullptr && gate_rows == T;
  const int groups = gate == nullptr || token_gate ? 1 : gate_rows;
  const int per = ctas_per_group(T, D, groups);
  const long long rows = (long long)groups * per;
  const bool z = post != nullptr || (gate != nullptr && !token_gate);
  if (rows > 0x7fffffffll || parts_floats < rows * D * (z ? 2 : 1)) return -1;
  NormArgs a = {};
  a.x = x; a.y = y; a.weight = weight; a.post = post; a.gate = gate;
  a.rstd = const_cast<float*>(rstd);
  a.dh = dh; a.dn = dn;
  a.dx = dx; a.dy = dy; a.dgate = dgate;
  a.w_parts = parts;
  a.z_parts = z ? parts + rows * D : nullptr;
  a.T = T; a.D = D;
  a.scale = scale;
  a.group_rows = T / groups;
  a.ctas_per_group = per;
  a.token_gate = token_gate ? 1 : 0;
  ParamArgs p = {};
  p.w_parts = a.w_parts; p.z_parts = a.z_parts;
  p.post = post; p.gate = gate;
  p.dw = dw; p.dpost = dpost; p.dgate = token_gate ? nullptr : dgate;
  p.dw_kind = dw_kind; p.dpost_kind = dpost_kind;
  p.dw_sumsq = dw_sumsq; p.dpost_sumsq = dpost_sumsq;
  p.scale = scale;
  p.D = D;
  p.groups = groups; p.ctas_per_group = per;
  p.token_gate = token_gate ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == 0 ? bwd_launch<__nv_bfloat16>(a, p, st) : dtype == 1 ? bwd_launch<__half>(a, p, st) : bwd_launch<float>(a, p, st);
}
