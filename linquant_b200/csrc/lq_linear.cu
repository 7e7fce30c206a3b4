// INT8 matrix product with a scale per token and per output channel.
//
//   y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n]          INT32 sums, exact
//
// Kernel for few tokens, where the weights' bytes and latency count: a CTA owns 16 output channels and up to 8 MT tokens. The rows
// of the weights come whole (2560 bytes of each at a time, two such pieces on their way) by bulk copies into shared memory; its
// warps share K in blocks of 64 bytes and add their INT32 sums through shared memory. The reduction index may be permuted as
// long as both operands are, so a lane takes 16 consecutive bytes of a row as the K slots of two m16n8k32 products. With values
// for codes (VALUES) every CTA makes the codes of its tokens in shared memory while the weights are on their way.
// 3 tokens, 5120 -> 2560 channels: fragments loaded straight from global memory, 64 bytes of a row at a time, took 8.2 us, and
// 11.5 us with a kernel for the codes ahead of it.
#include "lq_layer.cuh"
#include "lq_tc.cuh"

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
  constexpr int R = 8;  // rows at a time: their loads are on their way together
  const int tid = threadIdx.x, warp = tid >> 5;
  float top[R] = {};
#pragma unroll 2
  for (int c = tid * PV; c < K; c += THREADS * PV) {
    Pack<T, PV> raw[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < rows) raw[r] = load_pack<T, PV>(in + r * stride + c);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= rows) break;
      float v[PV];
      raw[r].get(v);
#pragma unroll
      for (int i = 0; i < PV; ++i) top[r] = max_nan(top[r], fabsf(v[i]));
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
#pragma unroll
    for (int m = 16; m; m >>= 1) top[r] = max_nan(top[r], __shfl_xor_sync(0xffffffffu, top[r], m));
    if ((tid & 31) == 0) part[r * 32 + warp] = top[r];
  }
  __syncthreads();
  float inv[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
    float amax = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) amax = max_nan(amax, part[r * 32 + w]);
    const float scale = row_scale(amax, inv[r]);
    if (tid == 0) scales[r] = scale;
  }
  for (int c = tid * PV; c < pitch; c += THREADS * PV) {
    Pack<T, PV> raw[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      raw[r].zero();
      if (r < rows && c < K) raw[r] = load_pack<T, PV>(in + r * stride + c);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= rows) break;
      float v[PV];
      raw[r].get(v);
      Pack<int8_t, PV> q;
      if constexpr (PV % 4 == 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
        for (int i = 0; i < PV; i += 4)
          w[i / 4] = pack_sat_s8x2(row_code(v[i + 1], inv[r]), row_code(v[i], inv[r]), pack_sat_s8x2(row_code(v[i + 3], inv[r]), row_code(v[i + 2], inv[r]), 0u));
      } else {
        q.v[0] = (int8_t)row_code(v[0], inv[r]);
      }
      store_pack(codes + r * pitch + c, q);
    }
  }
  __syncthreads();
}

constexpr int KC = 2560, WP = KC + 64;  // bytes of K at a time; pitch of a row of weights in shared memory (two rows of an access on banks of their own)

static __host__ __device__ __forceinline__ int code_pitch(int K) {  // of codes in shared memory: blocks of 64, an odd number of them
  const int p = (K + 63) / 64 * 64;
  return p % 128 ? p : p + 64;
}

template <int MT, typename TO, typename TX, int PV>
__global__ void __launch_bounds__(std::is_same_v<TX, int8_t> ? 256 : 512) int8_linear_few_kernel(const lq_linear_problem p, const Values values) {
  constexpr bool VALUES = !std::is_same_v<TX, int8_t>;
  constexpr int WARPS = VALUES ? 16 : 8;  // making codes takes instructions
  extern __shared__ __align__(128) int8_t dyn[];
  __shared__ int part[WARPS][8 * MT][17];
  __shared__ float scales[8 * MT], amax[VALUES ? 8 * 32 : 1];
  __shared__ uint64_t bars[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * MT;
  const int chunks = (p.K + KC - 1) / KC, K16 = p.K & ~15;
  int8_t* codes = dyn + (chunks > 1 ? 2 : 1) * 16 * WP;
  const int pitch = code_pitch(p.K);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(smem_u32(&bars[i])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  pdl_enter();
  auto request = [&](int c) {  // warp 0: one row a lane
    const int bytes = min(KC, K16 - c * KC);
    const uint32_t bar = smem_u32(&bars[c & 1]);
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((uint32_t)(bytes > 0 ? 16 * bytes : 0)) : "memory");
    __syncwarp();
    if (lane < 16 && bytes > 0) {
      const int8_t* from = p.w + (long long)min(n0 + lane, p.N - 1) * p.w_stride + (long long)c * KC;  // rows behind the last are read and not written
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dyn + ((c & 1) * 16 + lane) * WP)),
                   "l"(from), "r"(bytes), "r"(bar)
                   : "memory");
    }
  };
  if (warp == 0) {
    __syncwarp();
    request(0);
    if (chunks > 1) request(1);
  }
  if constexpr (VALUES)
    quantize_rows_shared<TX, PV, 32 * WARPS>(reinterpret_cast<const TX*>(values.x) + (long long)m0 * values.stride, values.stride, min(8, p.M - m0), p.K, codes, pitch, scales, amax);
  else
    __syncthreads();  // the barriers are there
  const int8_t* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = VALUES ? codes + min(g, p.M - m0 - 1) * pitch : p.x + (long long)min(m0 + 8 * j + g, p.M - 1) * p.x_stride;
  int acc[MT][4] = {};
  bool ok = true;
  for (int c = 0; c < chunks; ++c) {
    int8_t* w = dyn + (c & 1) * 16 * WP;
    if (c == chunks - 1 && K16 < p.K && tid < 16) {  // what is left of a row behind its last 16 bytes
      const int8_t* from = p.w + (long long)min(n0 + tid, p.N - 1) * p.w_stride;
      for (int k = K16; k < p.K; ++k) w[tid * WP + k - c * KC] = from[k];
    }
    const int k0 = c * KC, blocks = min(KC / 64, (p.K - k0 + 63) / 64);
    constexpr int U = (KC / 64 + WARPS - 1) / WARPS;
    uint4 b[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + (warp + u * WARPS) * 64 + 16 * q;
#pragma unroll
      for (int j = 0; j < MT; ++j) b[u][j] = !VALUES ? codes16(xr[j], k, p.K) : k < pitch ? *reinterpret_cast<const uint4*>(xr[j] + k) : make_uint4(0, 0, 0, 0);
    }
    ok = ok && mbar_wait_bounded(smem_u32(&bars[c & 1]), (uint32_t)((c >> 1) & 1));
    if (c == chunks - 1) __syncthreads();  // the ends of the rows
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = warp + u * WARPS;
      if (kb >= blocks) break;
      const uint4 lo = *reinterpret_cast<const uint4*>(w + g * WP + kb * 64 + 16 * q), hi = *reinterpret_cast<const uint4*>(w + (g + 8) * WP + kb * 64 + 16 * q);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        mma_s8(acc[j], lo.x, hi.x, lo.y, hi.y, b[u][j].x, b[u][j].y);
        mma_s8(acc[j], lo.z, hi.z, lo.w, hi.w, b[u][j].z, b[u][j].w);
      }
    }
    if (c + 2 < chunks) {
      __syncthreads();
      if (warp == 0) {
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        request(c + 2);
      }
    }
  }
  if (!ok && p.status) atomicExch(p.status, 1);
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][8 * j + 2 * q + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
  ok = __syncthreads_and(ok) != 0;
  if (!ok) {  // stores nothing; what was requested still lands
    for (int c = max(0, chunks - 2); c < chunks; ++c) mbar_wait_bounded(smem_u32(&bars[c & 1]), (uint32_t)((c >> 1) & 1));
    return;
  }
  for (int i = tid; i < 8 * MT * 16; i += 32 * WARPS) {
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
static int launch_few(const lq_linear_problem* p, const Values& v, cudaStream_t st) {
  const dim3 grid((p->N + 15) / 16, (p->M + 8 * MT - 1) / (8 * MT));
  const size_t smem = (size_t)(p->K > KC ? 2 : 1) * 16 * WP + (std::is_same_v<TX, int8_t> ? 0 : (size_t)(p->M < 8 ? p->M : 8) * code_pitch(p->K));
  const cudaError_t e = launch_opt_in(int8_linear_few_kernel<MT, TO, TX, PV>, grid, dim3(std::is_same_v<TX, int8_t> ? 256 : 512), smem, st, *p, v);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "int8_linear: %s", cudaGetErrorString(e));
  return check_launch("int8_linear_few_kernel");
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
  if (p->M > 16) return run_linear_tc(p, st);  // 5120 -> 2560 channels: 8 tokens 5.9 us here, 16 10.1, there 11.7 (8.4 from 32 on)
  return with_dtype(p->out_dtype, "int8_linear", [&](auto t) {
    using TO = decltype(t);
    return p->M <= 8 ? linear::launch_few<1, TO, int8_t, 1>(p, {}, st) : linear::launch_few<2, TO, int8_t, 1>(p, {}, st);
  });
}

extern "C" int lq_int8_linear_values(const lq_linear_problem* p, const void* values, int dtype, long long stride, lq_stream stream) {
  using namespace lq;
  if (int e = linear::check(p)) return e;
  if (dtype < LQ_F16 || dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "int8_linear_values: dtype %d", dtype);
  if (p->M == 0) return LQ_OK;
  if (!values) return fail(LQ_ERR_NULL, "int8_linear_values: values is null");
  cudaStream_t st = (cudaStream_t)stream;
  // up to eight tokens whose codes fit a CTA's shared memory next to the weights
  if (p->M > 8 || (long long)p->M * linear::code_pitch(p->K) > 128 * 1024) {
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
      return wide ? linear::launch_few<1, TO, TX, FULL>(p, v, st) : linear::launch_few<1, TO, TX, 1>(p, v, st);
    });
  });
}
