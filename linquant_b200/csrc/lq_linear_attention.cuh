// What the two kernels of linear attention share: the decays of a chunk, pieces of fp32 values, segments of a call's tokens.
#pragma once
#include "lq_layer.cuh"
#include "lq_tc.cuh"

namespace lq {

namespace attention {

__device__ __forceinline__ void sts_v4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void lds_v4(uint32_t addr, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(lds_u32(addr)); }
__device__ __forceinline__ float2 lds_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <typename T>
struct Half {  // the 16-bit type of the products
  using type = T;
};
template <>
struct Half<float> {
  using type = __nv_bfloat16;
};
// fp32 pairs as N pairs of pieces, the largest first
template <typename M, int N>
__device__ __forceinline__ void split(float a, float b, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = Act<M>::pack2(a, b);
    if (i + 1 < N) a -= Act<M>::get(p[i], 0), b -= Act<M>::get(p[i], 1);
  }
}
// 2^n, n cut to what a normal float holds
__device__ __forceinline__ float pow2(int n) { return __int_as_float((min(max(n, -126), 127) + 127) << 23); }
// n with 2^n <= m < 2^(n+1); 0 for zero, infinities and NaN
__device__ __forceinline__ int exponent(float m) {
  const int e = (__float_as_int(m) >> 23) & 255;
  return e == 0 || e == 255 ? 0 : e - 127;
}

struct Segments {
  int count, tokens;  // of a segment: a multiple of 64
  float* states;      // [count - 1][B * H][V tiles][floats of a tile]: what leaves a segment
  float* decays;      // [count - 1][B * H]: log2 of a segment's decay, which may leave fp32 itself
};

// The log-decays of a chunk's tokens from t0, C / 32 a lane; none behind the sequence's n tokens
template <int C>
__device__ __forceinline__ void load_decay(float (&x)[C / 32], const lq_attention_problem& p, int b, int h, int t0, int n) {
  const int lane = threadIdx.x & 31;
  const float* g = p.g + b * p.g_stride_b + h * p.g_stride_h;
#pragma unroll
  for (int i = 0; i < C / 32; ++i) {
    const int t = t0 + lane * (C / 32) + i;
    x[i] = p.g != nullptr && t < n ? __ldg(g + t * p.g_stride_t) : 0.f;
  }
}
// a value as the sum of two floats, the second at most half a step of the first
struct Pair {
  float hi = 0.f, lo = 0.f;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float h, float l) : hi(h), lo(l) {}
  __device__ __forceinline__ Pair operator+(const Pair& o) const {
    const float s = __fadd_rn(hi, o.hi), b = __fsub_rn(s, hi);
    const float e = __fadd_rn(__fadd_rn(__fsub_rn(hi, __fsub_rn(s, b)), __fsub_rn(o.hi, b)), __fadd_rn(lo, o.lo)), h = __fadd_rn(s, e);
    return Pair(h, __fsub_rn(e, __fsub_rn(h, s)));
  }
};

// One warp: the chunk's running sums of g in units of log2, and the decays that follow from them. A step below -128 is one of -128: its
// exponential is zero in fp32 either way, and the sums stay finite behind a step of minus infinity.
template <int C>
struct Decay {
  static constexpr int PER = C / 32, BYTES = (3 * C + 4) * 4;  // on a 16-byte boundary again
  float hi[PER], lo[PER], out[PER], all;  // of this lane's tokens; of the whole chunk
  // Sums of two floats each: a step of the scan is a dozen dependent fp32 additions, where one in 64 bits takes several times as long
  __device__ __forceinline__ Pair of(const float (&x)[PER]) {
    const int lane = threadIdx.x & 31;
    Pair sum[PER], run;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float g = x[i] < -128.f ? -128.f : x[i], p = g * kLog2e;
      const Pair step(p, fmaf(g, kLog2e, -p) + g * 1.92596299e-8f);  // log2(e) = a float and what it leaves
      sum[i] = run = i ? run + step : step;
    }
    Pair before = run;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const Pair o(__shfl_up_sync(0xffffffffu, before.hi, m), __shfl_up_sync(0xffffffffu, before.lo, m)), both = before + o;
      if (lane >= m) before = both;
    }
    const Pair total(__shfl_sync(0xffffffffu, before.hi, 31), __shfl_sync(0xffffffffu, before.lo, 31));
    const Pair first(__shfl_up_sync(0xffffffffu, before.hi, 1), __shfl_up_sync(0xffffffffu, before.lo, 1));  // what the lanes before have
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const Pair s = lane ? first + sum[i] : sum[i];
      hi[i] = s.hi;
      lo[i] = s.lo;
      out[i] = ex2((total.hi - s.hi) + (total.lo - s.lo));
    }
    all = ex2(total.hi);
    return total;
  }
  // running sums, what they lost to rounding, decays to the chunk's end; its whole decay
  __device__ __forceinline__ void store(uint32_t s_g) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t to = s_g + 4 * (lane * PER + i);
      sts_u32(to, __float_as_uint(hi[i]));
      sts_u32(to + 4 * C, __float_as_uint(lo[i]));
      sts_u32(to + 8 * C, __float_as_uint(out[i]));
    }
    if (lane == 0) sts_u32(s_g + 12 * C, __float_as_uint(all));
  }
};

// The decayed products of one warp's 16 rows (fragments of m16n8: columns 8 j + 2 t4, rows g and g + 8 from r0) with NJ tiles of
// columns, zero above the diagonal. Differences of sums high and low: exact where the sums are large.
template <int C, int NJ>
__device__ __forceinline__ void decay_products(float (&a)[NJ][4], uint32_t s_g, int r0, int tiles) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const float hi0 = lds_f32(s_g + 4 * (r0 + g)), hi1 = lds_f32(s_g + 4 * (r0 + g + 8));
  const float lo0 = lds_f32(s_g + 4 * (C + r0 + g)), lo1 = lds_f32(s_g + 4 * (C + r0 + g + 8));
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (j >= tiles) break;
    const int col = 8 * j + 2 * t4;
    const float2 hi = lds_f2(s_g + 4 * col), lo = lds_f2(s_g + 4 * (C + col));
    a[j][0] = col <= r0 + g ? a[j][0] * ex2((hi0 - hi.x) + (lo0 - lo.x)) : 0.f;
    a[j][1] = col + 1 <= r0 + g ? a[j][1] * ex2((hi0 - hi.y) + (lo0 - lo.y)) : 0.f;
    a[j][2] = col <= r0 + g + 8 ? a[j][2] * ex2((hi1 - hi.x) + (lo1 - lo.x)) : 0.f;
    a[j][3] = col + 1 <= r0 + g + 8 ? a[j][3] * ex2((hi1 - hi.y) + (lo1 - lo.y)) : 0.f;
  }
}
// fp16: the powers of two under which the rows g and g + 8 stay in the type's range
template <int NJ>
__device__ __forceinline__ void row_scales(const float (&a)[NJ][4], int tiles, float& up0, float& up1) {
  float top0 = 0.f, top1 = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (j >= tiles) break;
    top0 = fmaxf(top0, fmaxf(fabsf(a[j][0]), fabsf(a[j][1])));
    top1 = fmaxf(top1, fmaxf(fabsf(a[j][2]), fabsf(a[j][3])));
  }
#pragma unroll
  for (int m = 1; m < 4; m <<= 1) {
    top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, m));
    top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, m));
  }
  up0 = pow2(min(14 - exponent(top0), 40));
  up1 = pow2(min(14 - exponent(top1), 40));
}

// lq_linear_attention_tc.cu: the kernel for many tokens of 16-bit operands on tcgen05, where it applies
bool tc_applies(const lq_attention_problem* p);
struct Plan {
  int floats, count, tokens;  // of a state's tile; segments and their tokens
  long long tiles;          // B * H * V tiles
  bool tc;
};
int run_tc(const lq_attention_problem* p, const Plan& r, const Segments& seg, cudaStream_t st);
cudaError_t launch_segment_states(const Segments& seg, int heads, long long values, cudaStream_t st);

}  // namespace attention

}  // namespace lq
