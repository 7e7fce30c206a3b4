// INT8 matrix product with a scale per token and per output channel.
//
//   y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n]          INT32 sums, exact
//
// Warp-level kernel for few tokens, where the weights' bytes and latency count: a CTA owns 16 output channels and up to 8 MT
// tokens, its warps share K in blocks of 64 bytes and add their INT32 sums through shared memory. Weights go from global memory
// straight into MMA fragments: the reduction index may be permuted as long as both operands are, so a lane takes 16 consecutive
// bytes of a row as the K slots of two m16n8k32 products. All blocks of a warp are requested at once where K allows (five); with
// values for codes (VALUES) every CTA then makes the codes of its own tokens in shared memory while the weights are on their
// way: a kernel of its own for that took 3 us before the first weight was requested.
#include "lq_layer.cuh"

namespace lq {

namespace linear {

__device__ __forceinline__ uint4 ldg16(const int8_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// bytes [k, k + 16) of a row of K codes, zero from K on
__device__ __forceinline__ uint4 codes16(const int8_t* row, int k, int K) {
  if (k >= K) return make_uint4(0, 0, 0, 0);
  uint4 v = ldg16(row + k);
  const int left = K - k;
  if (left < 16) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = left - 4 * i;
      w[i] = n <= 0 ? 0u : n >= 4 ? w[i] : w[i] & (0xffffffffu >> (32 - 8 * n));
    }
  }
  return v;
}

struct Values {
  const void* x;
  long long stride;
};

// The codes of rows [0, rows) of `in` at pitch `pitch` in shared memory (zeros from K on) and their scales. PV values a load.
template <typename T, int PV, int THREADS>
__device__ __forceinline__ void quantize_rows_shared(const T* in, long long stride, int rows, int K, int8_t* codes, int pitch, float* scales, float* part) {
  const int tid = threadIdx.x, warp = tid >> 5;
  for (int r = 0; r < rows; ++r) {
    const T* row = in + r * stride;
    float amax = 0.f;
    for (int c = tid * PV; c < K; c += THREADS * PV) {
      float v[PV];
      load_pack<T, PV>(row + c).get(v);
#pragma unroll
      for (int i = 0; i < PV; ++i) amax = max_nan(amax, fabsf(v[i]));
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    if ((tid & 31) == 0) part[r * 32 + warp] = amax;
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    float amax = 0.f, inv;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) amax = max_nan(amax, part[r * 32 + w]);
    const float scale = row_scale(amax, inv);
    if (tid == 0) scales[r] = scale;
    const T* row = in + r * stride;
    for (int c = tid * PV; c < pitch; c += THREADS * PV) {
      int8_t q[PV] = {};
      if (c < K) {
        float v[PV];
        load_pack<T, PV>(row + c).get(v);
#pragma unroll
        for (int i = 0; i < PV; ++i) q[i] = (int8_t)q8(v[i], inv, 127.f);
      }
      store_pack(codes + r * pitch + c, *reinterpret_cast<Pack<int8_t, PV>*>(q));
    }
  }
  __syncthreads();
}

template <int MT, typename TO, int WARPS, typename TX, int PV>
__global__ void __launch_bounds__(32 * WARPS) int8_linear_warp_kernel(const lq_linear_problem p, const Values values) {
  pdl_enter();
  constexpr bool VALUES = !std::is_same_v<TX, int8_t>;
  constexpr int U = MT == 1 ? 5 : MT == 2 ? 4 : 2;  // K blocks requested at a time
  extern __shared__ __align__(16) int8_t dyn[];
  __shared__ int part[WARPS][8 * MT][17];
  __shared__ float scales[8 * MT], amax[VALUES ? 8 * 32 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * MT;
  const int nlo = min(n0 + g, p.N - 1), nhi = min(n0 + g + 8, p.N - 1);  // rows behind the last are read and not written
  const int8_t *wlo = p.w + nlo * p.w_stride, *whi = p.w + nhi * p.w_stride;
  const int blocks = (p.K + 63) / 64, pitch = blocks * 64 + 16;
  uint4 a[U][2];
  auto request = [&](int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (kb + u * WARPS) * 64 + 16 * q;
      a[u][0] = codes16(wlo, k, p.K);
      a[u][1] = codes16(whi, k, p.K);
    }
  };
  request(warp);
  if constexpr (VALUES)
    quantize_rows_shared<TX, PV, 32 * WARPS>(reinterpret_cast<const TX*>(values.x) + (long long)m0 * values.stride, values.stride, min(8, p.M - m0), p.K, dyn, pitch, scales, amax);
  const int8_t* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = VALUES ? dyn + min(g, p.M - m0 - 1) * pitch : p.x + (long long)min(m0 + 8 * j + g, p.M - 1) * p.x_stride;
  int acc[MT][4] = {};
  for (int kb = warp; kb < blocks; kb += U * WARPS) {
    uint4 b[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (kb + u * WARPS) * 64 + 16 * q;
#pragma unroll
      for (int j = 0; j < MT; ++j) b[u][j] = !VALUES ? codes16(xr[j], k, p.K) : k < pitch - 16 ? *reinterpret_cast<const uint4*>(xr[j] + k) : make_uint4(0, 0, 0, 0);
    }
    if (kb != warp) request(kb);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        mma_s8(acc[j], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][j].x, b[u][j].y);
        mma_s8(acc[j], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][j].z, b[u][j].w);
      }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][8 * j + 2 * q + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * MT * 16; i += 32 * WARPS) {
    const int m = m0 + (i >> 4), n = n0 + (i & 15);
    if (m >= p.M || n >= p.N) continue;
    int s = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += part[w][i >> 4][i & 15];
    const float y = fmaf((float)s * (VALUES ? scales[i >> 4] : p.x_scale[m]), p.w_scale[n], p.bias ? p.bias[n] : 0.f);
    reinterpret_cast<TO*>(p.y)[(size_t)m * p.N + n] = from_f32<TO>(y);
  }
}

template <int MT, typename TO, typename TX, int PV>
static int launch_warp(const lq_linear_problem* p, const Values& v, cudaStream_t st) {
  const dim3 grid((p->N + 15) / 16, (p->M + 8 * MT - 1) / (8 * MT));
  const size_t smem = std::is_same_v<TX, int8_t> ? 0 : (size_t)(p->M < 8 ? p->M : 8) * ((p->K + 63) / 64 * 64 + 16);
  cudaError_t e;
  // Sixteen warps where there is K for them (five blocks of 64 each): one round of requests instead of two
  if (MT == 1 && p->K > 2560) {
    auto kern = int8_linear_warp_kernel<MT, TO, MT == 1 ? 16 : 8, TX, PV>;
    e = smem > 40000 ? launch_opt_in(kern, grid, dim3(512), smem, st, *p, v) : launch(kern, grid, dim3(512), smem, st, *p, v);
  } else {
    auto kern = int8_linear_warp_kernel<MT, TO, 8, TX, PV>;
    e = smem > 40000 ? launch_opt_in(kern, grid, dim3(256), smem, st, *p, v) : launch(kern, grid, dim3(256), smem, st, *p, v);
  }
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "int8_linear: %s", cudaGetErrorString(e));
  return check_launch("int8_linear_warp_kernel");
}

static int check(const lq_linear_problem* p) {
  if (!p) return fail(LQ_ERR_NULL, "int8_linear: problem descriptor is null");
  if (p->M < 0 || p->N <= 0 || p->K <= 0 || p->K > 131071) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d N=%d K=%d", p->M, p->N, p->K);
  if (p->out_dtype < LQ_F16 || p->out_dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "int8_linear: dtype %d", p->out_dtype);
  if (p->M == 0) return LQ_OK;
  if (!p->x || !p->w || !p->x_scale || !p->w_scale || !p->y) return fail(LQ_ERR_NULL, "int8_linear: x, w, their scales and y must be non-null");
  Alignment a;
  if (a.at(p->x).at(p->w).pitch(p->x_stride, 1).pitch(p->w_stride, 1).bytes() != 16)
    return fail(LQ_ERR_ALIGN, "int8_linear: rows of codes start on 16-byte boundaries (pitches %lld, %lld)", p->x_stride, p->w_stride);
  return LQ_OK;
}

}  // namespace linear

int run_linear_tc(const lq_linear_problem* p, cudaStream_t st);  // lq_linear_tc.cu

}  // namespace lq

extern "C" int lq_int8_linear(const lq_linear_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = linear::check(p)) return e;
  if (p->M == 0) return LQ_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->M > 16) return run_linear_tc(p, st);  // 5120 -> 2560 channels: 8 tokens 8 us here, 16 11, 32 15, there 13 up to 256
  return with_dtype(p->out_dtype, "int8_linear", [&](auto t) {
    using TO = decltype(t);
    return p->M <= 8 ? linear::launch_warp<1, TO, int8_t, 1>(p, {}, st) : linear::launch_warp<2, TO, int8_t, 1>(p, {}, st);
  });
}

extern "C" int lq_int8_linear_values(const lq_linear_problem* p, const void* values, int dtype, long long stride, lq_stream stream) {
  using namespace lq;
  if (int e = linear::check(p)) return e;
  if (dtype < LQ_F16 || dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "int8_linear_values: dtype %d", dtype);
  if (p->M == 0) return LQ_OK;
  if (!values) return fail(LQ_ERR_NULL, "int8_linear_values: values is null");
  cudaStream_t st = (cudaStream_t)stream;
  // up to eight tokens whose codes fit a CTA's shared memory next to another CTA's
  if (p->M > 8 || (long long)p->M * (p->K + 80) > 100 * 1024) {
    if (int e = lq_quantize_rows(values, dtype, p->M, p->K, stride, const_cast<int8_t*>(p->x), p->x_stride, const_cast<float*>(p->x_scale), stream)) return e;
    return lq_int8_linear(p, stream);
  }
  return with_dtype(dtype, "int8_linear_values", [&](auto x) {
    using TX = decltype(x);
    constexpr int FULL = 16 / sizeof(TX);
    Alignment a;
    const bool wide = a.at(values).pitch(stride, sizeof(TX)).pitch(p->K, sizeof(TX)).bytes() == 16;
    return with_dtype(p->out_dtype, "int8_linear_values", [&](auto t) {
      using TO = decltype(t);
      const linear::Values v{values, stride};
      return wide ? linear::launch_warp<1, TO, TX, FULL>(p, v, st) : linear::launch_warp<1, TO, TX, 1>(p, v, st);
    });
  });
}
