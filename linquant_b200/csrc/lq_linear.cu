// INT8 matrix product with a scale per token and per output channel.
//
//   y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n]          INT32 sums, exact
//
// Kernel for few tokens, where the weights' bytes and latency count: a CTA walks over tiles of 16 output channels for up to 8 MT
// tokens. The rows of the weights come whole (2560 bytes of each at a time, two such pieces on their way) by bulk copies into
// shared memory; its warps share K in blocks of 64 bytes and add their INT32 sums through shared memory. The reduction index may
// be permuted as long as both operands are, so a lane takes 16 consecutive bytes of a row as the K slots of two m16n8k32 products.
// With values for codes (VALUES) every CTA makes the codes of its tokens in shared memory while the weights are on their way.
// 5120 -> 2560 channels: 3 tokens 6.9 us (13 MB, 2 us of memory; launch, the first bytes' latency and the sums' way through shared
// memory are the rest), with values 9.1, with a kernel for the codes ahead 10.1; 2560 -> 10576: 8 tokens 9.2, with values 11.3.
// A CTA for every tile, each making its codes, took 21.5 there.
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

// The codes of up to 8 rows of `in` at pitch `pitch` in shared memory (zeros from K on) and their scales; PV values a load. A row
// belongs to a power of two of warps. A thread's first HOLD loads stay in registers, what lies behind them is read again.
template <typename T, int PV, int WARPS>
__device__ __forceinline__ void quantize_rows_shared(const T* in, long long stride, int rows, int K, int8_t* codes, int pitch, float* scales, float* part) {
  constexpr int HOLD = 6;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = WARPS / (rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8);
  const int row = warp / team, step = team * 32 * PV, c0 = (warp % team * 32 + lane) * PV;
  const bool on = row < rows;
  const T* from = in + row * stride;
  Pack<T, PV> held[HOLD];
  auto load = [&](int c) {
    Pack<T, PV> raw;
    raw.zero();
    if (on && c < K) raw = load_pack<T, PV>(from + c);
    return raw;
  };
  float top = 0.f;
  auto largest = [&](const Pack<T, PV>& raw) {
    float v[PV];
    raw.get(v);
#pragma unroll
    for (int i = 0; i < PV; ++i) top = max_nan(top, fabsf(v[i]));
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h) held[h] = load(c0 + h * step);
#pragma unroll
  for (int h = 0; h < HOLD; ++h) largest(held[h]);
  for (int c = c0 + HOLD * step; c < K; c += step) largest(load(c));
#pragma unroll
  for (int m = 16; m; m >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
  if (lane == 0) part[warp] = top;
  __syncthreads();
  for (int w = 0; w < team; ++w) top = max_nan(top, part[row * team + w]);
  float inv;
  const float scale = row_scale(top, inv);
  if (on && lane == 0 && warp % team == 0) scales[row] = scale;
  auto store = [&](int c, const Pack<T, PV>& raw) {
    if (!on || c >= pitch) return;
    float v[PV];
    raw.get(v);
    Pack<int8_t, PV> q;
    if constexpr (PV % 4 == 0) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
      for (int i = 0; i < PV; i += 4)
        w[i / 4] = pack_sat_s8x2(row_code(v[i + 1], inv), row_code(v[i], inv), pack_sat_s8x2(row_code(v[i + 3], inv), row_code(v[i + 2], inv), 0u));
    } else {
      q.v[0] = (int8_t)row_code(v[0], inv);
    }
    store_pack(codes + row * pitch + c, q);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h) store(c0 + h * step, held[h]);
  for (int c = c0 + HOLD * step; c < pitch; c += step) store(c, load(c));
  __syncthreads();
}

// Bytes of K at a time: two pieces of 16 rows, 82 KB, leave room for two CTAs an SM (one next to the longest codes, 120 KB),
// and 40 blocks of 64 are whole rounds for 8 warps. Rows of another length end in a shorter piece. WP: pitch of a row of weights in
// shared memory (two rows of an access on banks of their own).
constexpr int KC = 2560, WP = KC + 64;

static __host__ __device__ __forceinline__ int code_pitch(int K) {  // of codes in shared memory: blocks of 64, an odd number of them
  const int p = (K + 63) / 64 * 64;
  return p % 128 ? p : p + 64;
}

template <int MT, typename TO, typename TX, int PV>
__global__ void __launch_bounds__(std::is_same_v<TX, int8_t> ? 256 : 512, 2) int8_linear_few_kernel(const lq_linear_problem p, const Values values) {
  constexpr bool VALUES = !std::is_same_v<TX, int8_t>;
  constexpr int WARPS = VALUES ? 16 : 8;  // making codes takes instructions
  extern __shared__ __align__(128) int8_t dyn[];
  __shared__ int part[WARPS][8 * MT][17];
  __shared__ float scales[8 * MT], amax[WARPS];
  __shared__ uint64_t bars[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int tiles = (p.N + 15) / 16, chunks = (p.K + KC - 1) / KC, K16 = p.K & ~15;
  const int items = ((tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x) * chunks;  // pieces of weights, one after the other
  int8_t* codes = dyn + 2 * 16 * WP;
  const int pitch = code_pitch(p.K);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(smem_u32(&bars[i])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  pdl_enter();
  struct At {  // of an item: its tile and piece
    int tile, chunk;
    __device__ __forceinline__ void next(int chunks) {
      if (++chunk == chunks) chunk = 0, tile += gridDim.x;
    }
  };
  auto request = [&](int item, const At& at) {  // warp 0: one row a lane
    const int bytes = max(0, min(KC, K16 - at.chunk * KC));
    const uint32_t bar = smem_u32(&bars[item & 1]);
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((uint32_t)(16 * bytes)) : "memory");
    __syncwarp();
    if (lane < 16 && bytes > 0) {
      const int8_t* from = p.w + (long long)min(at.tile * 16 + lane, p.N - 1) * p.w_stride + (long long)at.chunk * KC;  // rows behind the last are read and not written
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(dyn + ((item & 1) * 16 + lane) * WP)),
                   "l"(from), "r"(bytes), "r"(bar)
                   : "memory");
    }
  };
  At ahead{(int)blockIdx.x, 0};
  for (int i = 0; i < 2 && i < items; ++i, ahead.next(chunks))
    if (warp == 0) request(i, ahead);
  // thread tid stores output (tid / 16, tid % 16) of a tile; its scales and bias are requested ahead
  static_assert(8 * MT * 16 <= 32 * WARPS);
  const int m = tid >> 4;
  const bool mine = m < p.M;
  const float xs = !VALUES && mine ? __ldg(p.x_scale + m) : 0.f;
  if constexpr (VALUES)
    quantize_rows_shared<TX, PV, WARPS>(reinterpret_cast<const TX*>(values.x), values.stride, p.M, p.K, codes, pitch, scales, amax);
  else
    __syncthreads();  // the barriers are there
  const int8_t* xr[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) xr[j] = VALUES ? codes + min(g, p.M - 1) * pitch : p.x + (long long)min(8 * j + g, p.M - 1) * p.x_stride;
  int acc[MT][4] = {};
  bool ok = true;
  At at{(int)blockIdx.x, 0};
  float ws = 0.f, bias = 0.f;
  for (int i = 0; i < items; ++i, at.next(chunks), ahead.next(chunks)) {
    int8_t* w = dyn + (i & 1) * 16 * WP;
    const int n0 = at.tile * 16, on = n0 + (tid & 15), k0 = at.chunk * KC, blocks = min(KC / 64, (p.K - k0 + 63) / 64);
    const bool last = at.chunk == chunks - 1;
    if (at.chunk == 0 && mine && on < p.N) {
      ws = __ldg(p.w_scale + on);
      bias = p.bias ? __ldg(p.bias + on) : 0.f;
    }
    constexpr int U = (KC / 64 + WARPS - 1) / WARPS;
    uint4 b[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + (warp + u * WARPS) * 64 + 16 * q;
#pragma unroll
      for (int j = 0; j < MT; ++j) b[u][j] = !VALUES ? codes16(xr[j], k, p.K) : k < pitch ? *reinterpret_cast<const uint4*>(xr[j] + k) : make_uint4(0, 0, 0, 0);
    }
    if (last && K16 < p.K) {  // what is left of a row behind its last 16 bytes
      if (tid < 16) {
        const int8_t* from = p.w + (long long)min(n0 + tid, p.N - 1) * p.w_stride;
        for (int k = K16; k < p.K; ++k) w[tid * WP + k - k0] = from[k];
      }
      __syncthreads();
    }
    ok = ok && mbar_wait_bounded(smem_u32(&bars[i & 1]), (uint32_t)((i >> 1) & 1));
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
    if (last) {
      if (chunks == 1 && i > 0) __syncthreads();  // the sums of the tile before have been read
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[warp][8 * j + 2 * q + (e & 1)][g + 8 * (e >> 1)] = acc[j][e], acc[j][e] = 0;
    }
    ok = __syncthreads_and(ok) != 0;
    if (!ok) {  // stores nothing more; what was requested still lands
      for (int k = i; k < min(i + 2, items); ++k) mbar_wait_bounded(smem_u32(&bars[k & 1]), (uint32_t)((k >> 1) & 1));
      if (tid == 0 && p.status) atomicExch(p.status, 1);
      return;
    }
    if (warp == 0 && i + 2 < items) {
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      request(i + 2, ahead);
    }
    if (last && mine && on < p.N) {
      int s = 0;
#pragma unroll
      for (int v = 0; v < WARPS; ++v) s += part[v][m][tid & 15];
      reinterpret_cast<TO*>(p.y)[(size_t)m * p.N + on] = from_f32<TO>(fmaf((float)s * (VALUES ? scales[m] : xs), ws, bias));
    }
  }
}

constexpr int CODES = 120 * 1024;  // bytes of codes that a CTA makes at most, next to the weights

// The opt-in to shared memory is a kernel's most and not what a call needs: it belongs to the kernel on its device, and another
// thread's smaller call between this one's opt-in and its launch would have the launch refused.
template <int MT, typename TO, typename TX, int PV>
static int launch_few(const lq_linear_problem* p, const Values& v, cudaStream_t st) {
  constexpr bool VALUES = !std::is_same_v<TX, int8_t>;
  constexpr int most_smem = 2 * 16 * WP + (VALUES ? CODES : 0);
  const size_t smem = 2 * 16 * WP + (VALUES ? (size_t)p->M * code_pitch(p->K) : 0);
  auto kern = int8_linear_few_kernel<MT, TO, TX, PV>;
  const int threads = VALUES ? 512 : 256;
  int per_sm = 0;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
  if (e == cudaSuccess) {
    const int tiles = (p->N + 15) / 16, most = sm_count() * per_sm;
    e = launch(kern, dim3(tiles < most ? tiles : most), dim3(threads), smem, st, *p, v);
  }
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "int8_linear: %s", cudaGetErrorString(e));
  return check_launch("int8_linear_few_kernel");
}

static int check(const lq_linear_problem* p) {
  if (!p) return fail(LQ_ERR_NULL, "int8_linear: problem descriptor is null");
  if (p->M < 0 || p->N <= 0 || p->K <= 0 || p->K > 131071 || !fits(p->M) || !fits(p->N)) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d N=%d K=%d", p->M, p->N, p->K);
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
  if (p->M > 16) return run_linear_tc(p, st);  // 5120 -> 2560 channels: 8 tokens 7.0 us here, 16 9.5, there 11.7 (7.9 from 32 on)
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
  // up to eight tokens whose codes fit a CTA's shared memory next to the weights: one launch, and 8.1 us against 9.5 (1 token), 10.8
  // against 10.2 (5), 11.3 against 10.2 (8) at 5120 -> 2560, where the host's 2 us for another launch are not counted
  if (p->M > 8 || (long long)p->M * linear::code_pitch(p->K) > linear::CODES) {
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
