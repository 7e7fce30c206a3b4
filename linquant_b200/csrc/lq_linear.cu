// INT8 matrix product with a scale per token and per output channel.
//
//   y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n]          INT32 sums, exact
//
// Warp-level kernel: a CTA owns 16 output channels and up to 8 MT tokens, its eight warps share K in blocks of 64 bytes and
// add their INT32 sums through shared memory. Weights and codes go from global memory straight into MMA fragments: the
// reduction index may be permuted as long as both operands are, so a lane takes 16 consecutive bytes of a row as the K slots
// of two m16n8k32 products.
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

constexpr int WARPS = 8;

template <int MT, typename TO>
__global__ void __launch_bounds__(32 * WARPS) int8_linear_warp_kernel(const lq_linear_problem p) {
  pdl_enter();
  constexpr int U = MT <= 2 ? 4 : 2;  // K blocks requested at a time
  __shared__ int part[WARPS][8 * MT][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * MT;
  const int nlo = min(n0 + g, p.N - 1), nhi = min(n0 + g + 8, p.N - 1);  // rows behind the last are read and not written
  const int8_t *wlo = p.w + nlo * p.w_stride, *whi = p.w + nhi * p.w_stride;
  const int8_t* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = p.x + (long long)min(m0 + 8 * j + g, p.M - 1) * p.x_stride;
  int acc[MT][4] = {};
  const int blocks = (p.K + 63) / 64;
  for (int kb = warp; kb < blocks; kb += U * WARPS) {
    uint4 a[U][2], b[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (kb + u * WARPS) * 64 + 16 * q;
      a[u][0] = codes16(wlo, k, p.K);
      a[u][1] = codes16(whi, k, p.K);
#pragma unroll
      for (int j = 0; j < MT; ++j) b[u][j] = codes16(xr[j], k, p.K);
    }
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
    const float y = fmaf((float)s * p.x_scale[m], p.w_scale[n], p.bias ? p.bias[n] : 0.f);
    reinterpret_cast<TO*>(p.y)[(size_t)m * p.N + n] = from_f32<TO>(y);
  }
}

template <int MT, typename TO>
static int launch_warp(const lq_linear_problem* p, cudaStream_t st) {
  const dim3 grid((p->N + 15) / 16, (p->M + 8 * MT - 1) / (8 * MT));
  if (grid.y > 65535) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d", p->M);
  launch(int8_linear_warp_kernel<MT, TO>, grid, dim3(32 * WARPS), 0, st, *p);
  return check_launch("int8_linear_warp_kernel");
}

}  // namespace linear

int run_linear_tc(const lq_linear_problem* p, cudaStream_t st);  // lq_linear_tc.cu

}  // namespace lq

extern "C" int lq_int8_linear(const lq_linear_problem* p, lq_stream stream) {
  using namespace lq;
  if (!p) return fail(LQ_ERR_NULL, "int8_linear: problem descriptor is null");
  if (p->M < 0 || p->N <= 0 || p->K <= 0 || p->K > 131071) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d N=%d K=%d", p->M, p->N, p->K);
  if (p->out_dtype < LQ_F16 || p->out_dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "int8_linear: dtype %d", p->out_dtype);
  if (p->M == 0) return LQ_OK;
  if (!p->x || !p->w || !p->x_scale || !p->w_scale || !p->y) return fail(LQ_ERR_NULL, "int8_linear: x, w, their scales and y must be non-null");
  Alignment a;
  if (a.at(p->x).at(p->w).pitch(p->x_stride, 1).pitch(p->w_stride, 1).bytes() != 16)
    return fail(LQ_ERR_ALIGN, "int8_linear: rows of codes start on 16-byte boundaries (pitches %lld, %lld)", p->x_stride, p->w_stride);
  cudaStream_t st = (cudaStream_t)stream;
  if (p->M > 64) return run_linear_tc(p, st);
  return with_dtype(p->out_dtype, "int8_linear", [&](auto t) {
    using TO = decltype(t);
    return p->M <= 8 ? linear::launch_warp<1, TO>(p, st) : p->M <= 16 ? linear::launch_warp<2, TO>(p, st) : linear::launch_warp<4, TO>(p, st);
  });
}
