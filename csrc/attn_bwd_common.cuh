// What the two attention backward kernels have in common around their main kernel: the order of the CTAs, the parts of a key tile, the pre-pass and
// the post-pass.
#pragma once
#include "common.cuh"

namespace {

constexpr int HD = 128;
constexpr int BQ = 64;    // query rows per step
constexpr int BKV = 128;  // keys per CTA

YF_DEVINL void tma_reduce_add_3d(const CUtensorMap* m, const void* smem_src, int x, int y, int z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// Where a CTA that shares its key tile leaves dK (is_v = 0) and dV: [head_parts][B][key tiles][Hkv][2] blocks of 32 groups of four head
// dims x 128 keys, so that a warp, one key per lane, stores 512 contiguous bytes at a time (rows of 128 dims: 16 bytes in each of
// 32 lines).
constexpr int PART_TILE = BKV * HD / 4;  // float4s of a block
__host__ __device__ inline long long part_tile(int part, int B, int b, int n_kt, int jt, int Hkv, int hk, int is_v) {
  return (((((long long)part * B + b) * n_kt + jt) * Hkv + hk) * 2 + is_v) * PART_TILE;
}

// Order of the CTAs: heads are taken in groups, within a group key tile by key tile with the heads fastest, so that all heads'
// long walks start first.  One group holds all heads unless the dQ accumulator outgrows the L2 and there are heads for three
// groups; then a group has two CTAs per SM, whose sums stay in the L2.  It pays for many sequences or long ones: 8 x 2048 tokens x 32
// heads 1449 us in one group, 1247 in groups of 19; 2 x 8192 x 32 3516 / 3438 in groups of five; 2 x 2304 x 32 393 / 380; 2 x 4096 x
// 32 971 / 995 in groups of ten; 1 x 4096 x 64 984 / 1013.  1 x 8192 x 32/8 stays whole: 1543 us, 1572 in two groups.
YF_DEVINL void head_group_order(int cta, int n_pos, int n_heads, int group, int& pos, int& head) {
  const int per_group = n_pos * group;
  const int g = cta / per_group;
  const int r = cta - g * per_group;
  const int size = min(group, n_heads - g * group);
  pos = r / size;
  head = g * group + r - pos * size;
}
int head_group_size(int n_pos, int n_heads, long long accum_bytes, int n_sms) {
  const int group = (2 * n_sms + n_pos - 1) / n_pos;
  return accum_bytes <= (64ll << 20) || group >= n_heads / 3 ? n_heads : group;
}

// delta[b,h,s] = sum_d dO * O, and the fp32 dQ accumulator of the same (token, head) cleared on the way (the main kernel
// adds into it): sixteen lanes per (token, head), one 16-byte load of O and of dO and two 16-byte stores of zeros per lane.
// LO: O is the sum of two bf16 tensors (what rounding it to bf16 left over is kept, see attn_mods.cuh).
template <bool LO>
__global__ void __launch_bounds__(256) attn_delta_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ o_lo, const __nv_bfloat16* __restrict__ d_o,
                                                         float* __restrict__ delta, float* __restrict__ dq_zero, int B, int S, int Hq,
                                                         long long o_stride, long long do_stride) {
  const long long total = (long long)B * S * Hq;
  const int sub = threadIdx.x & 15;
  const unsigned half_mask = 0xffffu << (threadIdx.x & 16);  // the two halves of a warp may leave the loop at different times
  for (long long w = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 4; w < total;
       w += ((long long)gridDim.x * blockDim.x) >> 4) {
    const int h = (int)(w % Hq);
    const long long t = w / Hq;
    const uint4 a = *reinterpret_cast<const uint4*>(o + t * o_stride + h * HD + sub * 8);
    const uint4 g = *reinterpret_cast<const uint4*>(d_o + t * do_stride + h * HD + sub * 8);
    if (dq_zero != nullptr) {
      float4* z = reinterpret_cast<float4*>(dq_zero + (t * Hq + h) * HD + sub * 8);
      z[0] = make_float4(0.f, 0.f, 0.f, 0.f);
      z[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float2 a0 = unpack_bf16x2(a.x), a1 = unpack_bf16x2(a.y), a2 = unpack_bf16x2(a.z), a3 = unpack_bf16x2(a.w);
    const float2 g0 = unpack_bf16x2(g.x), g1 = unpack_bf16x2(g.y), g2 = unpack_bf16x2(g.z), g3 = unpack_bf16x2(g.w);
    float s = a0.x * g0.x + a0.y * g0.y + a1.x * g1.x + a1.y * g1.y + a2.x * g2.x + a2.y * g2.y + a3.x * g3.x + a3.y * g3.y;
    if (LO) {
      const uint4 l = *reinterpret_cast<const uint4*>(o_lo + t * o_stride + h * HD + sub * 8);
      const float2 l0 = unpack_bf16x2(l.x), l1 = unpack_bf16x2(l.y), l2 = unpack_bf16x2(l.z), l3 = unpack_bf16x2(l.w);
      s += l0.x * g0.x + l0.y * g0.y + l1.x * g1.x + l1.y * g1.y + l2.x * g2.x + l2.y * g2.y + l3.x * g3.x + l3.y * g3.y;
    }
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(half_mask, s, m);
    if (sub == 0) {
      const long long bb = t / S, ss = t % S;
      delta[(bb * Hq + h) * S + ss] = s;
    }
  }
}

// dst, dst + 64 (bf16) = f * (a, z): eight head dims and their partners 64 further on.  With `cs` (cos, sin of the eight dims) they
// go back through the rotation on the way.
YF_DEVINL void store_gradient(__nv_bfloat16* dst, float (&a)[8], float (&z)[8], const float4* cs, float f) {
  if (cs != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 c = __ldg(cs + j);
      const float a0 = a[2 * j], a1 = a[2 * j + 1];
      a[2 * j] = a0 * c.x + z[2 * j] * c.y;
      a[2 * j + 1] = a1 * c.z + z[2 * j + 1] * c.w;
      z[2 * j] = z[2 * j] * c.x - a0 * c.y;
      z[2 * j + 1] = z[2 * j + 1] * c.z - a1 * c.w;
    }
  }
  uint4 w;
  w.x = pack_bf16x2(a[0] * f, a[1] * f); w.y = pack_bf16x2(a[2] * f, a[3] * f);
  w.z = pack_bf16x2(a[4] * f, a[5] * f); w.w = pack_bf16x2(a[6] * f, a[7] * f);
  *reinterpret_cast<uint4*>(dst) = w;
  w.x = pack_bf16x2(z[0] * f, z[1] * f); w.y = pack_bf16x2(z[2] * f, z[3] * f);
  w.z = pack_bf16x2(z[4] * f, z[5] * f); w.w = pack_bf16x2(z[6] * f, z[7] * f);
  *reinterpret_cast<uint4*>(dst + 64) = w;
}
YF_DEVINL const float4* rope_at(const float* rope, int pos, int dim) {
  return rope == nullptr ? nullptr : reinterpret_cast<const float4*>(rope + ((long long)pos * 64 + dim) * 2);
}

// Whether token t, the i-th of its sequence of S, sees one key only; spans null: causal.  Its probability is 1 whatever q and k are, so they get no
// gradient from it: zeros, not what is left of the difference of two equal sums.
YF_DEVINL bool sees_one_key(const int2* spans, long long t, int i, int S) {
  if (spans == nullptr) return i == 0;
  const int2 s = __ldg(spans + t);
  return min(s.y, S) - max(s.x, 0) == 1;
}

// dq (bf16, strided rows) = scale * dq_accum (fp32, dense rows of 128 Hq); with dkv_parts also dk = scale * the sum of the parts' dK and
// dv = that of their dV, in the order of the parts.  RANGES: rows of dq that see one key are zeros.  `rope` ([S, 64, 2]: cos, sin): dq and dk go back through the rotation.
template <bool RANGES>
__global__ void __launch_bounds__(256) attn_convert_kernel(const float* __restrict__ dq_acc, const float4* __restrict__ dkv_parts, int parts, const float* __restrict__ rope,
                                    __nv_bfloat16* __restrict__ dq, __nv_bfloat16* __restrict__ dk, __nv_bfloat16* __restrict__ dv, int B,
                                    int S, int Hq, int Hkv, long long dq_stride, long long dkv_stride, float scale, const int2* __restrict__ spans) {
  const long long first = blockIdx.x * (long long)blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
  const long long n_dq = (long long)B * S * Hq * 8;
  const int n_kt = (S + BKV - 1) / BKV;
  const long long blocks = dkv_parts == nullptr ? 0 : (long long)B * n_kt * Hkv * 2;  // of a part
  const long long total = n_dq + blocks * (BKV * 8);
  for (long long i = first; i < total; i += step) {
    float a[8], z[8];
    if (i < n_dq) {
      const long long t = i / (Hq * 8);
      const int u = (int)(i - t * (Hq * 8)), h = u >> 3, v = (u & 7) * 8;
      const float4* src = reinterpret_cast<const float4*>(dq_acc + (t * Hq + h) * HD + v);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 x = src[j], y = src[16 + j];
        a[4 * j] = x.x; a[4 * j + 1] = x.y; a[4 * j + 2] = x.z; a[4 * j + 3] = x.w;
        z[4 * j] = y.x; z[4 * j + 1] = y.y; z[4 * j + 2] = y.z; z[4 * j + 3] = y.w;
      }
      if (RANGES && sees_one_key(spans, t, (int)(t % S), S)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = z[j] = 0.f;
      }
      store_gradient(dq + t * dq_stride + h * HD + v, a, z, rope_at(rope, (int)(t % S), v), scale);
    } else {  // a warp: eight keys x four groups of dims (whole lines read, 64 contiguous bytes per key written)
      const long long k = i - n_dq, block = k >> 10;
      const int v = ((int)k & 3) + ((int)(k >> 5) & 1) * 4, row = ((int)(k >> 2) & 7) + ((int)(k >> 6) & 15) * 8, is_v = (int)(block & 1);
      const long long bj = (block >> 1) / Hkv;
      const int hk = (int)((block >> 1) - bj * Hkv), s = (int)(bj % n_kt) * BKV + row;
      if (s >= S) continue;
      const float4* src = dkv_parts + block * PART_TILE + 2 * v * BKV + row;
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = z[j] = 0.f;
      for (int p0 = 0; p0 < parts; p0 += 4, src += 4 * blocks * PART_TILE) {  // four parts in flight
        float4 x[4][4];
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[p][j] = p0 + p < parts ? __ldcg(src + p * blocks * PART_TILE + ((j & 1) + (j >> 1) * 16) * BKV) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            a[4 * j] += x[p][j].x; a[4 * j + 1] += x[p][j].y; a[4 * j + 2] += x[p][j].z; a[4 * j + 3] += x[p][j].w;
            z[4 * j] += x[p][2 + j].x; z[4 * j + 1] += x[p][2 + j].y; z[4 * j + 2] += x[p][2 + j].z; z[4 * j + 3] += x[p][2 + j].w;
          }
      }
      __nv_bfloat16* dst = (is_v ? dv : dk) + ((bj / n_kt) * S + s) * dkv_stride + hk * HD + v * 8;
      store_gradient(dst, a, z, is_v ? nullptr : rope_at(rope, s, v * 8), is_v ? 1.f : scale);
    }
  }
}

}  // namespace
