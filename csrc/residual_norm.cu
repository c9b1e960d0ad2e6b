// The residual step between two blocks of a decoder for sm_100a:
//   u = y * rsqrt(mean(y^2) + eps) * post      (the norm after the block; u = y without one)
//   h = x + scale * gate * u                    (gate: none, one row for a group of tokens, or a row per token)
//   n = h * rsqrt(mean(h^2) + eps) * weight     (the norm before the next block)
// and its gradients.  With dh, dn the gradients of h and n, and hats for what a norm has divided:
//   g = dh + r_h (dn weight - hhat mean(dn weight hhat)) = dx
//   e = scale gate g,  dy = r_y (e post - yhat mean(e post yhat)),
//   dweight = sum dn hhat,  dpost = sum e yhat,  dgate = scale sum g u  over the tokens that share the row.
// Bound by HBM: forward reads x, y and writes h, n once; backward reads x, y, dh, dn and writes dx, dy once.  h is formed anew in
// the backward pass: the rounded h would take as many bytes and lose bits.  All sums are fp32, in a fixed order.
#include "common.cuh"
#include "vec8.cuh"
#include "yafsdp_b200.h"

namespace {

constexpr int NV = 2;  // vectors of 8 per thread: TPR threads hold a row of up to 16 TPR elements

template <int TPR>
constexpr int BLOCK = TPR < 256 ? 256 : TPR;

// sum over the TPR threads of a row.  `slots`: one float per warp of the block, not used again before the row's threads have met at another
// barrier.
template <int TPR>
YF_DEVINL float row_sum(float v, float* slots, int group) {
  v = warp_sum(v);
  if (TPR == 32) return v;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  if (TPR >= 256) __syncthreads();
  else if (group == 0) named_bar_sync(1, TPR);  // literal barrier numbers: a computed one reserves all sixteen
  else if (group == 1) named_bar_sync(2, TPR);
  else if (group == 2) named_bar_sync(3, TPR);
  else named_bar_sync(4, TPR);
  v = 0.f;
#pragma unroll
  for (int g = 0; g < TPR / 32; ++g) v += slots[group * (TPR / 32) + g];
  return v;
}

struct NormArgs {
  const void *x, *y, *weight, *post, *gate;  // post, gate: may be null
  void *h, *n;
  float* rstd;  // [T, 2]: r_y (with post), r_h; may be null
  const void *dh, *dn;  // either may be null: zeros
  void *dx, *dy, *dgate;
  float *w_parts, *z_parts;  // [CTAs, D]: sums of dn hhat and of g yhat (g y without post; e yhat with a gate per token)
  float scale, eps;
  int T, D;
  int group_rows;    // tokens that share a row of the gate (1: a gate per token)
  int ctas_per_group;
};

template <typename T, int TPR>
__global__ void __launch_bounds__(BLOCK<TPR>) residual_norm_fwd_kernel(NormArgs a) {
  constexpr int ROWS = BLOCK<TPR> / TPR;
  __shared__ float slots[2][BLOCK<TPR> / 32];
  const int group = threadIdx.x / TPR, tr = threadIdx.x % TPR;
  const int row = blockIdx.x * ROWS + group;
  if (row >= a.T) return;
  const long long at = (long long)row * a.D;
  const T* x = reinterpret_cast<const T*>(a.x) + at;
  const T* y = reinterpret_cast<const T*>(a.y) + at;
  const T* gate = reinterpret_cast<const T*>(a.gate) + (a.gate ? (long long)(row / a.group_rows) * a.D : 0);
  const T *post = reinterpret_cast<const T*>(a.post), *w = reinterpret_cast<const T*>(a.weight);
  const int nvec = a.D / 8;
  float h[NV][8], u[NV][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tr + TPR * i;
    if (v < nvec) {
      load_f8<T>(x + v * 8, h[i]);
      load_f8<T>(y + v * 8, u[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += u[i][j] * u[i][j];
    }
  }
  float ry = 1.f;
  if (a.post) ry = rsqrtf(row_sum<TPR>(ss, slots[0], group) / (float)a.D + a.eps);
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tr + TPR * i;
    if (v < nvec) {
      float f[8], s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = a.scale;
      if (a.gate) {
        load_f8<T>(gate + v * 8, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] *= f[j];
      }
      if (a.post) {
        load_f8<T>(post + v * 8, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[i][j] *= ry * f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[i][j] += s[j] * u[i][j];
        ss += h[i][j] * h[i][j];
      }
      store_f8<T>(reinterpret_cast<T*>(a.h) + at + v * 8, h[i]);
    }
  }
  const float rh = rsqrtf(row_sum<TPR>(ss, slots[1], group) / (float)a.D + a.eps);
  if (tr == 0 && a.rstd) reinterpret_cast<float2*>(a.rstd)[row] = make_float2(ry, rh);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tr + TPR * i;
    if (v < nvec) {
      float f[8];
      load_f8<T>(w + v * 8, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= h[i][j] * rh;
      store_f8<T>(reinterpret_cast<T*>(a.n) + at + v * 8, f);
    }
  }
}

// A CTA walks over the rows of one group of tokens (all tokens where the gate is per token); its threads hold the same columns of every
// row and sum the parameters' gradients in registers on the way.
template <typename T, int TPR, bool TOKEN_GATE>
__global__ void __launch_bounds__(BLOCK<TPR>) residual_norm_bwd_kernel(NormArgs a) {
  constexpr int THREADS = BLOCK<TPR>, ROWS = THREADS / TPR;
  __shared__ float slots[2][2][THREADS / 32];
  __shared__ float sums[ROWS > 1 ? TPR * NV * 8 : 1];
  const int group = threadIdx.x / TPR, tr = threadIdx.x % TPR;
  const int nvec = a.D / 8;
  const int part = blockIdx.x % a.ctas_per_group, gg = blockIdx.x / a.ctas_per_group;
  const int rows = TOKEN_GATE ? a.T : a.group_rows;
  const float inv_d = 1.f / (float)a.D;
  const T *post = reinterpret_cast<const T*>(a.post), *w = reinterpret_cast<const T*>(a.weight);
  const T* gate = reinterpret_cast<const T*>(a.gate) + (a.gate && !TOKEN_GATE ? (long long)gg * a.D : 0);
  float acc_w[NV][8], acc_z[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc_w[i][j] = acc_z[i][j] = 0.f;
  int parity = 0;
  for (int r = part * ROWS + group; r < rows; r += a.ctas_per_group * ROWS, parity ^= 1) {
    const long long row = (long long)gg * rows + r, at = row * a.D;
    const T *x = reinterpret_cast<const T*>(a.x) + at, *y = reinterpret_cast<const T*>(a.y) + at;
    const T *dh = reinterpret_cast<const T*>(a.dh) + (a.dh ? at : 0), *dn = reinterpret_cast<const T*>(a.dn) + (a.dn ? at : 0);
    const T* gr = gate + (TOKEN_GATE ? at : 0);
    const float2 rs = reinterpret_cast<const float2*>(a.rstd)[row];
    const float ry = rs.x, rh = rs.y;
    float yv[NV][8], hv[NV][8], g[NV][8], cv[NV][8], s[NV][8];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        float f[8];
        load_f8<T>(x + v * 8, hv[i]);
        load_f8<T>(y + v * 8, yv[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          yv[i][j] *= ry;  // yhat (y itself without post)
          s[i][j] = a.scale;
          g[i][j] = cv[i][j] = 0.f;
        }
        if (a.gate) {
          load_f8<T>(gr + v * 8, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[i][j] *= f[j];
        }
        if (a.dh) load_f8<T>(dh + v * 8, g[i]);
        if (a.dn) load_f8<T>(dn + v * 8, cv[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 1.f;
        if (a.post) load_f8<T>(post + v * 8, f);
        float wf[8];
        load_f8<T>(w + v * 8, wf);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hv[i][j] = (hv[i][j] + s[i][j] * (yv[i][j] * f[j])) * rh;  // hhat
          acc_w[i][j] += cv[i][j] * hv[i][j];
          cv[i][j] *= wf[j];
          dot += cv[i][j] * hv[i][j];
        }
      }
    }
    dot = row_sum<TPR>(dot, slots[0][parity], group) * inv_d;
    float dot2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[i][j] += rh * (cv[i][j] - hv[i][j] * dot);
          f[j] = 1.f;
        }
        store_f8<T>(reinterpret_cast<T*>(a.dx) + at + v * 8, g[i]);
        if (a.post) load_f8<T>(post + v * 8, f);
        float dg[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float gy = g[i][j] * yv[i][j];
          if (TOKEN_GATE) {
            dg[j] = a.scale * gy * f[j];
            acc_z[i][j] += s[i][j] * gy;
          } else {
            acc_z[i][j] += gy;
          }
          cv[i][j] = s[i][j] * g[i][j] * f[j];  // e post
          dot2 += cv[i][j] * yv[i][j];
        }
        if (TOKEN_GATE) store_f8<T>(reinterpret_cast<T*>(a.dgate) + at + v * 8, dg);
      }
    }
    if (a.post) dot2 = row_sum<TPR>(dot2, slots[1][parity], group) * inv_d;
    else dot2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tr + TPR * i;
      if (v < nvec) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = ry * (cv[i][j] - yv[i][j] * dot2);
        store_f8<T>(reinterpret_cast<T*>(a.dy) + at + v * 8, o);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* parts = k == 0 ? a.w_parts : a.z_parts;
    if (parts == nullptr) continue;
    float(&acc)[NV][8] = k == 0 ? acc_w : acc_z;
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
        if (v < nvec) store_f8<float>(parts + (long long)blockIdx.x * a.D + v * 8, acc[i]);
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
    dpost = finish(dpost);
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
  while (t * NV * 8 < D) t *= 2;
  return t;
}
// CTAs that walk over one group of tokens: two per SM altogether, no more than there are rows for
int ctas_per_group(int T, int D, int groups) {
  const int tpr = row_threads(D), rows = tpr < 256 ? 256 / tpr : 1, in_group = T / groups;
  int want = (2 * yf_num_sms() + groups - 1) / groups;
  const int most = (in_group + rows - 1) / rows;
  if (want > most) want = most;
  return want < 1 ? 1 : want;
}

template <typename T>
int fwd_launch(const NormArgs& a, cudaStream_t st) {
  const int tpr = row_threads(a.D);
#define YF_LAUNCH(N)                                                                                              \
  case N: {                                                                                                       \
    constexpr int rows = BLOCK<N> / N;                                                                  \
    residual_norm_fwd_kernel<T, N><<<(a.T + rows - 1) / rows, BLOCK<N>, 0, st>>>(a);                    \
    break;                                                                                                        \
  }
  switch (tpr) {
    YF_LAUNCH(32) YF_LAUNCH(64) YF_LAUNCH(128) YF_LAUNCH(256) YF_LAUNCH(512) YF_LAUNCH(1024)
    default: return -1;
  }
#undef YF_LAUNCH
  return -(int)cudaGetLastError();
}
template <typename T>
int bwd_launch(const NormArgs& a, const ParamArgs& p, cudaStream_t st) {
  const int tpr = row_threads(a.D), grid = p.groups * p.ctas_per_group;
#define YF_LAUNCH(N)                                                                                              \
  case N:                                                                                                         \
    if (p.token_gate) residual_norm_bwd_kernel<T, N, true><<<grid, BLOCK<N>, 0, st>>>(a);               \
    else residual_norm_bwd_kernel<T, N, false><<<grid, BLOCK<N>, 0, st>>>(a);                           \
    break;
  switch (tpr) {
    YF_LAUNCH(32) YF_LAUNCH(64) YF_LAUNCH(128) YF_LAUNCH(256) YF_LAUNCH(512) YF_LAUNCH(1024)
    default: return -1;
  }
#undef YF_LAUNCH
  residual_norm_param_kernel<T><<<(a.D + 31) / 32, 1024, 0, st>>>(p);
  return -(int)cudaGetLastError();
}

bool misaligned(const void* const* p, int n) {
  uintptr_t bits = 0;
  for (int i = 0; i < n; ++i) bits |= reinterpret_cast<uintptr_t>(p[i]);
  return (bits & 15) != 0;
}
bool bad_shape(int T, int D, int gate_rows, const void* gate, int dtype) {
  if (T <= 0 || D <= 0 || D % 8 || D > 16384 || dtype < 0 || dtype > 2) return true;
  return gate != nullptr ? gate_rows <= 0 || T % gate_rows != 0 : gate_rows != 0;
}

}  // namespace

// x, y, h, n: [T, D] without gaps; weight, post: [D]; gate: [gate_rows, D], row t / (T / gate_rows) for token t (gate_rows 0 without one); all
// of one type (dtype 0 bf16, 1 fp16, 2 fp32), 16-byte aligned, D a multiple of 8 up to 16384.  rstd: [T, 2] fp32 for the backward
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == 0 ? fwd_launch<__nv_bfloat16>(a, st) : dtype == 1 ? fwd_launch<__half>(a, st) : fwd_launch<float>(a, st);
}

// Rows of [rows, D] fp32 scratch that the backward pass wants (twice that with a post norm or a gate).
extern "C" int yf_residual_norm_parts(int T, int D, int gate_rows) {
  if (T <= 0 || D <= 0 || D % 8 || D > 16384 || gate_rows < 0 || (gate_rows > 0 && T % gate_rows)) return -1;
  const int groups = gate_rows == 0 || gate_rows == T ? 1 : gate_rows;
  const long long n = (long long)groups * ctas_per_group(T, D, groups);
  return n > 0x7fffffff ? -1 : (int)n;
}

// Gradients of yf_residual_norm_fwd.  dh, dn: either may be null (zeros).  parts: yf_residual_norm_parts rows of D floats, twice as many with
// post or gate; parts_floats says how many there are.  dw, dpost: kind 0 the type of the activations, 1 fp32, 2 fp32 that is added to;
// *_sumsq (optional): += the squares of what was written.
extern "C" int yf_residual_norm_bwd(const void* x, const void* y, const void* weight, const void* post, const void* gate, int gate_rows,
                                    const float* rstd, const void* dh, const void* dn, void* dx, void* dy, void* dw, int dw_kind, float* dw_sumsq,
                                    void* dpost, int dpost_kind, float* dpost_sumsq, void* dgate, float* parts, long long parts_floats, int T, int D,
                                    float scale, int dtype, void* stream) {
  const void* ptrs[] = {x, y, weight, post, gate, rstd, dh, dn, dx, dy, dgate, parts};
  if (bad_shape(T, D, gate_rows, gate, dtype) || !x || !y || !weight || !rstd || !dx || !dy || !dw || !parts || misaligned(ptrs, 12)) return -1;
  if ((post != nullptr) != (dpost != nullptr) || (gate != nullptr) != (dgate != nullptr)) return -1;
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
