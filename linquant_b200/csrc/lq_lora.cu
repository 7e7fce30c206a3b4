// INT8 product with low-rank adapters of many requests at once.
//
//   y[m,n] = (sum_k c[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n] + sum_r t[m,r] b[l,n,r],   t[m,r] = scaling[l] sum_k x[m,k] a[l,r,k]
//
// l = adapters[m]; c are x's codes. This file's first kernel makes t. Up to 16 tokens the INT8 product's kernel adds the second sum to its own in
// fp32 (lq_lora.cuh). For more this file's second kernel leaves it in fp32 scratch (for fp32 outputs in y itself) and the product's kernels add it
// from there, to the sum that is then rounded once. What runs beside the tcgen05 product on an SM's tensor cores waits for them (warp products in its epilogue: 510 us where the product alone takes 302, at
// 16384 x 2560 -> 10576 with rank 16; fp32 products there: 680).
// t: a CTA has a tile of 1, 8 or 16 tokens and, of a cluster, a part of K; its four warps share that part and their sums meet in
// shared memory, first the warps', then the CTAs', in a fixed order. Operands come from global memory straight into the fragments
// of m16n8k16 (the reduction index permuted alike in both: a lane takes eight consecutive k). A tile whose tokens have several
// adapters goes over its K once for each of them. Products are exact: both operands as bf16 pieces (codes and bf16 one, fp16 two, fp32
// three; codes or fp16 with fp16 as they are), six products for fp32.
// Both kernels let their successors start at once (pdl_trigger()): the product's loads and sums run beside them, and wait for t or the share where
// it is added. 3 tokens, 5120 -> 2560, rank 16: 11.4 us in a row, 15.6 without, 9.3 the product alone.
// 16384 tokens, 2560 -> 10576, rank 16: 514 us in a row, the product alone 310. t of 333 x 2560 codes, rank 32, 24 adapters in runs of 7: 11 us, bound by latency, a tile's adapters one after the other; of 16384 x 2560, rank 16:
// 22 us (42 MB of codes from HBM or L2, half of the issue slots).
#include "lq_lora.cuh"
#include "lq_tc.cuh"

namespace lq {

namespace lora {

constexpr int WARPS = 4, THREADS = 32 * WARPS;

template <typename TX, typename TA>
struct Types {
  static constexpr bool F16 = std::is_same_v<TA, __half> && (std::is_same_v<TX, __half> || std::is_same_v<TX, int8_t>);
  template <typename T>
  static constexpr int pieces() { return F16 ? 1 : sizeof(T) == 4 ? 3 : std::is_same_v<T, __half> ? 2 : 1; }
  static constexpr int NX = pieces<TX>(), NA = pieces<TA>(), KEEP = NX > NA ? NX : NA;
};

// Eight consecutive values, on their way and then as words of pairs in pieces. VEC: they start on a boundary of eight values (16 bytes at most)
template <typename T, bool VEC>
struct Eight {
  static constexpr int WORDS = VEC ? 2 * sizeof(T) : 8;
  uint32_t w[WORDS];
  // VEC: always read (a load behind a condition would have to land before the next one is issued); else what lies `left` values or more behind p is not
  __device__ __forceinline__ void load(const T* p, int left) {
    if constexpr (VEC && WORDS == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = 0.f;
        if (i < left) {
          if constexpr (std::is_same_v<T, int8_t>) x = (float)__ldg(p + i);
          else x = to_f32(p[i]);
        }
        w[i] = __float_as_uint(x);
      }
    }
  }
  __device__ __forceinline__ void keep(bool in) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = in ? w[i] : 0u;
  }
  template <int N, bool F16>
  __device__ __forceinline__ void pieces(uint32_t (&q)[N][4]) const {
    if constexpr (VEC && sizeof(T) == 2 && N == 1) {  // as they are
#pragma unroll
      for (int i = 0; i < 4; ++i) q[0][i] = w[i];
    } else {
      float x[8];
      if constexpr (VEC && std::is_same_v<T, int8_t>) {
        const uint32_t a = w[0] ^ 0x80808080u, b = w[1] ^ 0x80808080u;
        x[0] = s8_to_float<0>(a), x[1] = s8_to_float<1>(a), x[2] = s8_to_float<2>(a), x[3] = s8_to_float<3>(a);
        x[4] = s8_to_float<0>(b), x[5] = s8_to_float<1>(b), x[6] = s8_to_float<2>(b), x[7] = s8_to_float<3>(b);
      } else if constexpr (VEC && sizeof(T) == 2) {
        Act<T>::unpack8(make_uint4(w[0], w[1], w[2], w[3]), x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (F16) {
          q[0][i] = Act<__half>::pack2(x[2 * i], x[2 * i + 1]);
        } else {
          uint32_t r[N];
          bf16_pieces<N>(x[2 * i], x[2 * i + 1], r);
#pragma unroll
          for (int k = 0; k < N; ++k) q[k][i] = r[k];
        }
      }
    }
  }
};

struct Shrink {
  int M, K, L, R, RP, parts;
  long long x_stride;          // elements
  const void *x, *a;
  const float* x_scale;        // of codes, or null
  const int* adapters;
  const float* scaling;        // [L] or null
  float scale;
  int halves;                  // t as pieces: of four values their bf16 roundings, then those of what is left
  float* t;
};

// TILE: tokens of a CTA; NT: tiles of 8 ranks at a time
template <typename TX, typename TA, int TILE, bool VEC, int NT>
__global__ void __launch_bounds__(THREADS) lora_shrink_kernel(const Shrink p) {
  using Y = Types<TX, TA>;
  constexpr int MT = (TILE + 15) / 16, ROWS = 16 * MT;
  extern __shared__ __align__(16) float sums[];  // [WARPS][TILE][RP], then the CTA's own in the first
  __shared__ int which[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % p.parts, m0 = blockIdx.x / p.parts * TILE;
  pdl_enter();
  pdl_trigger();
  for (int i = tid; i < ROWS; i += THREADS) {
    const int l = i < TILE && m0 + i < p.M ? __ldg(p.adapters + m0 + i) : -1;
    which[i] = (unsigned)l < (unsigned)p.L ? l : -1;
  }
  for (int i = tid; i < WARPS * TILE * p.RP; i += THREADS) sums[i] = 0.f;
  __syncthreads();
  const int steps = (p.K + 31) / 32, step0 = (int)((long long)steps * rank / p.parts), step1 = (int)((long long)steps * (rank + 1) / p.parts);
  int l = -1;
  while (true) {
    // the next adapter of the tile, in rising order
    int next = 0x7fffffff;
    for (int i = lane; i < ROWS; i += 32)
      if (which[i] > l) next = min(next, which[i]);
    l = __reduce_min_sync(0xffffffffu, next);
    if (l == 0x7fffffff) break;
    for (int r0 = 0; r0 < p.R; r0 += 8 * NT) {
      const int tiles = min(NT, (p.R - r0) / 8);
      float acc[MT][NT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
      // what lies behind the last token, rank or channel is read from inside and made zero
      const TA* a[NT];
      const TX* x[MT][2];
      bool own[MT][2];  // a token with another adapter is zero for this one
#pragma unroll
      for (int j = 0; j < NT; ++j) a[j] = reinterpret_cast<const TA*>(p.a) + ((long long)l * p.R + min(r0 + 8 * j + g, p.R - 1)) * p.K;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * i + 8 * h + g;
          own[i][h] = which[row] == l;
          x[i][h] = reinterpret_cast<const TX*>(p.x) + (long long)(own[i][h] ? m0 + row : m0) * p.x_stride;
        }
      // U steps of 32 on their way
      constexpr int BYTES = MT * Eight<TX, VEC>::WORDS * 2 + NT * Eight<TA, VEC>::WORDS, U = BYTES <= 24 ? 4 : BYTES <= 48 ? 2 : 1;
      for (int s0 = step0 + warp; s0 < step1; s0 += U * WARPS) {
        Eight<TX, VEC> rx[U][MT][2];
        Eight<TA, VEC> ra[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = 32 * (s0 + u * WARPS) + 8 * t4, left = s0 + u * WARPS < step1 ? p.K - k : 0, at = VEC ? min(k, p.K - 8) : k;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) rx[u][i][h].load(x[i][h] + at, left);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (VEC || j < tiles) ra[u][j].load(a[j] + at, left);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool in = s0 + u * WARPS < step1 && p.K - 32 * (s0 + u * WARPS) - 8 * t4 > 0;
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) rx[u][i][h].keep(in && own[i][h]);
#pragma unroll
          for (int j = 0; j < NT; ++j) ra[u][j].keep(in && j < tiles);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t xa[MT][2][Y::NX][4];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) rx[u][i][h].template pieces<Y::NX, Y::F16>(xa[i][h]);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (j >= tiles) break;
            uint32_t b[Y::NA][4];
            ra[u][j].template pieces<Y::NA, Y::F16>(b);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int n = Y::NA - 1; n >= 0; --n)
#pragma unroll
                for (int o = Y::NX - 1; o >= 0; --o) {
                  if (n + o >= (Y::KEEP > 1 ? 3 : 1)) continue;
#pragma unroll
                  for (int i = 0; i < MT; ++i) {
                    if constexpr (Y::F16) mma_f16(acc[i][j], xa[i][0][o][2 * h], xa[i][1][o][2 * h], xa[i][0][o][2 * h + 1], xa[i][1][o][2 * h + 1], b[n][2 * h], b[n][2 * h + 1]);
                    else mma_bf16(acc[i][j], xa[i][0][o][2 * h], xa[i][1][o][2 * h], xa[i][0][o][2 * h + 1], xa[i][1][o][2 * h + 1], b[n][2 * h], b[n][2 * h + 1]);
                  }
                }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = 16 * i + g + 8 * (e >> 1), r = r0 + 8 * j + 2 * t4 + (e & 1);
            if (row < TILE && j < tiles && which[row] == l) sums[(warp * TILE + row) * p.RP + r] = acc[i][j][e];
          }
    }
  }
  __syncthreads();
  const int values = TILE * p.RP;
  for (int i = tid; i < values; i += THREADS) {
    float s = sums[i];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) s += sums[w * values + i];
    sums[i] = s;
  }
  if (p.parts > 1) cluster_sync();
  else __syncthreads();
  const uint32_t base = smem_u32(sums);
  for (int i = 4 * (rank * THREADS + tid); i < values; i += 4 * p.parts * THREADS) {  // four of a row
    const int row = i / p.RP, m = m0 + row;
    if (m >= p.M) continue;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < p.parts; ++c) {
      float4 v;
      uint32_t at = base + 4 * i;
      if (p.parts > 1) {
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(base + 4 * i), "r"(c));
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
      } else {
        v = *reinterpret_cast<const float4*>(sums + i);
      }
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const int own = which[row];
    if (own >= 0) {
      float f = p.scaling ? p.scale * __ldg(p.scaling + own) : p.scale;
      if (p.x_scale) f *= __ldg(p.x_scale + m);
      s.x *= f, s.y *= f, s.z *= f, s.w *= f;
    }
    uint4 w = make_uint4(__float_as_uint(s.x), __float_as_uint(s.y), __float_as_uint(s.z), __float_as_uint(s.w));
    if (p.halves) {
      uint32_t lo[2], hi[2];
      bf16_pieces<2>(s.x, s.y, lo);
      bf16_pieces<2>(s.z, s.w, hi);
      w = make_uint4(lo[0], hi[0], lo[1], hi[1]);
    }
    *reinterpret_cast<uint4*>(p.t + (long long)m * p.RP + i - row * p.RP) = w;
  }
  if (p.parts > 1) cluster_sync();  // no CTA's sums are read any more
}

template <typename TX, typename TA, int TILE, bool VEC, int NT>
static int shrink(const Shrink& p, int tiles, cudaStream_t st) {
  auto kern = lora_shrink_kernel<TX, TA, TILE, VEC, NT>;
  constexpr int most = WARPS * TILE * 128 * 4;
  cudaError_t e = cudaSuccess;
  if (most > 48 * 1024) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles * p.parts);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)WARPS * TILE * p.RP * 4;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = p.parts > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, p);
  }
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "lora_linear: %s", cudaGetErrorString(e));
  return check_launch("lora_shrink_kernel");
}

// Tokens of a CTA: one for few tokens, each of which may have an adapter of its own, as long as a's rows, read once for each, are few (100 x 2560
// of as many adapters, rank 16: 22 us where eight take 30; 256 x 5120 in runs of 7, rank 32: 36 and 27); eight up to four tokens an SM, whose
// tiles have fewer adapters to go through (333 tokens in runs of 7, rank 32: 34 us, 37 with sixteen); then sixteen (4000 tokens in runs of
// 500: 46 us, 49 with eight; 32 were no better). Parts of K: up to four CTAs an SM, and no fewer than 64 of K for a warp.
template <typename TX, typename TA>
static int run_shrink(Shrink p, bool vec, cudaStream_t st) {
  const int sms = sm_count(), tile = (long long)p.M * p.R <= 4096 ? 1 : p.M <= 4 * sms ? 8 : 16, tiles = (p.M + tile - 1) / tile;
  p.parts = 8;
  while (p.parts > 1 && ((long long)tiles * p.parts > 4ll * sms || p.K < 256 * p.parts)) p.parts /= 2;
  auto go = [&](auto v, auto nt) {
    constexpr bool VEC = decltype(v)::value;
    constexpr int NT = decltype(nt)::value;
    if (tile == 1) return shrink<TX, TA, 1, VEC, NT>(p, tiles, st);
    if (tile == 8) return shrink<TX, TA, 8, VEC, NT>(p, tiles, st);
    return shrink<TX, TA, 16, VEC, NT>(p, tiles, st);
  };
  auto width = [&](auto v) { return p.R <= 16 ? go(v, std::integral_constant<int, 2>()) : p.R <= 32 ? go(v, std::integral_constant<int, 4>()) : go(v, std::integral_constant<int, 8>()); };
  return vec ? width(std::true_type()) : width(std::false_type());
}

// ---- the second product: y[m,n] = sum_r t[m,r] b[l,n,r] for the tokens that have an adapter
constexpr int CHUNK = 32, CT = CHUNK / 8;  // channels at a time, in tiles of 8

// A warp: 16 MI tokens, SPAN channels; PT: pieces of t, two for 16-bit outputs and three for fp32. Over the adapters that the tokens have and their ranks in steps of 16; a step's operands are requested before
// the products of the one ahead. The reduction index is permuted alike in both operands: a lane takes four consecutive r; and the channels of
// a chunk, column 2 i + e of tile j being channel 8 i + 2 j + e, so that a lane holds eight consecutive ones of a row. Both operands are
// bf16 pieces: PT of t and of fp16 and fp32 b, products below 16 (24) bits behind the first left out.
// Many tokens: bound by the share's bytes (16384 x 10576, rank 16: 147 us, 4.7 TB/s). Few: by L2's latency.
template <int PT, typename TB, int SPAN, int MI>
__global__ void __launch_bounds__(THREADS, PT == 2 ? (MI == 1 ? 6 : 4) : 3) lora_expand_kernel(const Lora q, int M, int N) {
  constexpr int PB = std::is_same_v<TB, __nv_bfloat16> ? 1 : PT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int columns = (N + WARPS * SPAN - 1) / (WARPS * SPAN), m0 = (int)(blockIdx.x / columns) * (16 * MI), n0 = ((int)(blockIdx.x % columns) * WARPS + warp) * SPAN;
  if (n0 >= N) return;
  const int mine = lane < 16 * MI && m0 + lane < M ? q.of(m0 + lane) : -1;
  const uint32_t all = __ballot_sync(0xffffffffu, mine >= 0);
  const bool wide = PT == 2 || (N % 4 == 0 && (reinterpret_cast<uintptr_t>(q.share) & 15u) == 0);

  // the step that is on its way
  int l = 0, r0 = 0, c0 = 0;
  uint32_t rows = 0, left = 0;
  Pack<TB, 4> b[CT];
  uint4 t[MI][2];
  if (SPAN == 32) {  // few tokens: every adapter's rows of b on their way to L2, by its first one
    const uint32_t like = __match_any_sync(0xffffffffu, mine);
    const TB* from = reinterpret_cast<const TB*>(q.b) + ((long long)mine * N + n0) * q.R;
    if (mine >= 0 && (like & ((1u << lane) - 1)) == 0)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(from), "r"((uint32_t)(min(SPAN, N - n0) * q.R * (int)sizeof(TB))) : "memory");
  }
  pdl_enter();  // t; what ran before the kernel that makes it has completed
  pdl_trigger();
  if (!all) return;
  auto next_adapter = [&] {
    l = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
    rows = __ballot_sync(0xffffffffu, mine == l);
    left &= ~rows;
    r0 = 0;
  };
  auto request = [&] {
    const int r = r0 + 4 * t4, rb = min(r, q.R - 4);  // behind R t is zero, and b is made so
    const int n = n0 + c0 + 8 * (g >> 1) + (g & 1);
    if (n0 + c0 + CHUNK <= N) {
      const TB* from = reinterpret_cast<const TB*>(q.b) + ((long long)l * N + n) * q.R + rb;
#pragma unroll
      for (int j = 0; j < CT; ++j) b[j] = load_pack<TB, 4>(from + 2 * j * q.R);
    } else {  // behind N nothing is stored
#pragma unroll
      for (int j = 0; j < CT; ++j) b[j] = load_pack<TB, 4>(reinterpret_cast<const TB*>(q.b) + ((long long)l * N + min(n + 2 * j, N - 1)) * q.R + rb);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * i + 8 * h + g;  // of tokens with another adapter what comes of it is not kept
        t[i][h] = *reinterpret_cast<const uint4*>(q.t + (long long)min(m0 + row, M - 1) * q.RP + r);
      }
  };
  left = all;
  next_adapter();
  request();
  while (true) {
    const uint32_t now = rows;
    const int at = c0;
    float s[MI][CT][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][j][e] = 0.f;
    bool same = true, end = false;  // the adapter goes on; nothing is left
    while (same) {
      uint32_t a[MI][PT][4], w[CT][PB][2];
      const bool inside = r0 + 4 * t4 < q.R;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (PT == 2) {  // as the first kernel has left them
            a[i][0][h] = t[i][h].x, a[i][0][2 + h] = t[i][h].y, a[i][1][h] = t[i][h].z, a[i][1][2 + h] = t[i][h].w;
          } else {
            uint32_t lo[PT], hi[PT];
            bf16_pieces<PT>(__uint_as_float(t[i][h].x), __uint_as_float(t[i][h].y), lo);
            bf16_pieces<PT>(__uint_as_float(t[i][h].z), __uint_as_float(t[i][h].w), hi);
#pragma unroll
            for (int k = 0; k < PT; ++k) a[i][k][h] = lo[k], a[i][k][2 + h] = hi[k];
          }
        }
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        if constexpr (PB == 1) {
          const uint2 x = *reinterpret_cast<const uint2*>(&b[j]);
          w[j][0][0] = inside ? x.x : 0u, w[j][0][1] = inside ? x.y : 0u;
        } else {
          float x[4];
          b[j].get(x);
          uint32_t lo[PB], hi[PB];
          bf16_pieces<PB>(inside ? x[0] : 0.f, inside ? x[1] : 0.f, lo);
          bf16_pieces<PB>(inside ? x[2] : 0.f, inside ? x[3] : 0.f, hi);
#pragma unroll
          for (int k = 0; k < PB; ++k) w[j][k][0] = lo[k], w[j][k][1] = hi[k];
        }
      }
      r0 += 16;
      same = r0 < q.R;
      if (!same) {
        if (left == 0) {
          c0 += CHUNK;
          end = c0 >= SPAN || n0 + c0 >= N;
          left = all;
        }
        if (!end) next_adapter();
      }
      if (!end) request();
#pragma unroll
      for (int k = PB - 1; k >= 0; --k)
#pragma unroll
        for (int o = PT - 1; o >= 0; --o) {
          if (k + o >= PT) continue;
#pragma unroll
          for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) mma_bf16(s[i][j], a[i][o][0], a[i][o][1], a[i][o][2], a[i][o][3], w[j][k][0], w[j][k][1]);
        }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * i + 8 * h + g;
        if (!(now >> row & 1)) continue;
        const int n = n0 + at + 8 * t4;
#pragma unroll
        for (int c = 0; c < 8; c += 4) {
          const float4 x = make_float4(s[i][c / 2][2 * h], s[i][c / 2][2 * h + 1], s[i][c / 2 + 1][2 * h], s[i][c / 2 + 1][2 * h + 1]);
          float* to = PT == 2 ? q.share_at(m0 + row, n + c) : q.share + (size_t)(m0 + row) * N + n + c;
          if (wide) {
            if (n + c < N) *reinterpret_cast<float4*>(to) = x;
          } else {
            if (n + c < N) to[0] = x.x;
            if (n + c + 1 < N) to[1] = x.y;
            if (n + c + 2 < N) to[2] = x.z;
            if (n + c + 3 < N) to[3] = x.w;
          }
        }
      }
    if (end) return;
  }
}

static int expand(const Lora& q, const lq_linear_problem* p, cudaStream_t st) {
  return with_dtype(q.dtype, "lora_linear", [&](auto tb) {
    using TB = decltype(tb);
    auto pieces = [&](auto pt) {
      constexpr int PT = decltype(pt)::value;
      // Few tokens: warps of 16 of them and 32 channels, as many as there can be, each of which goes over all adapters of its tokens one after
      // the other (333 x 10576, rank 32, runs of 7: 40 us where the others' warps of 32 and 128 take 63; 1000 x 2560 25 and 27). Many: these
      // read b half as often (1000 x 10576, rank 16: 49 us and 54, 16384 tokens 519 and 595)
      auto go = [&](auto kern, int span, int tokens) {
        const long long rows = ((long long)p->M + tokens - 1) / tokens;
        const long long ctas = rows * ((p->N + WARPS * span - 1) / (WARPS * span));
        if (ctas >= 1ll << 31) return fail(LQ_ERR_SHAPE, "lora_linear: M=%d N=%d", p->M, p->N);
        const cudaError_t e = launch(kern, dim3((unsigned)ctas), dim3(THREADS), 0, st, q, p->M, p->N);
        return e != cudaSuccess ? fail(LQ_ERR_LAUNCH, "lora_linear: %s", cudaGetErrorString(e)) : check_launch("lora_expand_kernel");
      };
      return ((long long)p->M + 31) / 32 * ((p->N + 127) / 128) <= 10ll * sm_count() ? go(lora_expand_kernel<PT, TB, 32, 1>, 32, 16) : go(lora_expand_kernel<PT, TB, 128, 2>, 128, 32);
    };
    return p->out_dtype == LQ_F32 ? pieces(std::integral_constant<int, 3>()) : pieces(std::integral_constant<int, 2>());
  });
}

// 16-bit outputs of more than kFewTokens tokens: in slabs whose fp32 shares take about 1 GiB (and 1024 tokens at least), each made and added
// before the next one's. None has few tokens: they are of one size, but for the rounding to whole blocks of 32
struct Slabs {
  long long M, count, blocks;
  Slabs(int m, int N) : M(m), blocks(((long long)N + 3) / 4) {
    const long long most = (1ll << 26) / blocks < 1024 ? 1024 : (1ll << 26) / blocks;
    count = (M + most - 1) / most;
  }
  int start(long long i) const { return i >= count ? (int)M : (int)(M * i / count & ~31ll); }
  size_t bytes() const { return (size_t)(count == 1 ? (M + 31) / 32 : M / count / 32 + 2) * 32 * blocks * 16; }  // a slab: M / count + 31 tokens at most
};

}  // namespace lora

int run_linear(const lq_linear_problem* p, const Lora* lora, cudaStream_t st);                                              // lq_linear.cu
int run_linear_values(const lq_linear_problem* p, const Lora* lora, const void* values, int dtype, long long stride, cudaStream_t st);
int check_linear(const lq_linear_problem* p);
bool linear_makes_codes(const lq_linear_problem* p);

}  // namespace lq

extern "C" size_t lq_lora_workspace_bytes(int M, int R) { return M <= 0 || R <= 0 ? 0 : (size_t)M * ((R + 15) / 16 * 16) * 4; }
extern "C" size_t lq_lora_share_bytes(int M, int N, int out_dtype) {
  if (M <= lq::kFewTokens || N <= 0 || out_dtype == LQ_F32) return 0;
  return lq::lora::Slabs(M, N).bytes();
}

extern "C" int lq_lora_linear(const lq_linear_problem* p, const lq_lora_problem* q, const void* values, int dtype, long long stride, lq_stream stream) {
  using namespace lq;
  if (int e = check_linear(p)) return e;
  if (!q) return fail(LQ_ERR_NULL, "lora_linear: adapter descriptor is null");
  if (q->L < 0 || q->R <= 0 || !fits(q->L)) return fail(LQ_ERR_SHAPE, "lora_linear: L=%d R=%d", q->L, q->R);
  if (q->R % 8 || q->R > 128) return fail(LQ_ERR_UNSUPPORTED, "lora_linear: R=%d, multiples of 8 up to 128", q->R);
  if (q->dtype < LQ_F16 || q->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "lora_linear: dtype %d", q->dtype);
  if (values && (dtype < LQ_F16 || dtype > LQ_F32)) return fail(LQ_ERR_UNSUPPORTED, "lora_linear: dtype %d", dtype);
  if (p->M == 0) return LQ_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (q->L == 0) return values ? run_linear_values(p, nullptr, values, dtype, stride, st) : run_linear(p, nullptr, st);
  if (!q->a || !q->b || !q->adapters || !q->t) return fail(LQ_ERR_NULL, "lora_linear: a, b, adapters and t must be non-null");
  if ((reinterpret_cast<uintptr_t>(q->b) | reinterpret_cast<uintptr_t>(q->t)) & 15u) return fail(LQ_ERR_ALIGN, "lora_linear: b and t start on 16-byte boundaries");
  const int RP = (q->R + 15) / 16 * 16, size = dtype_bytes(q->dtype);
  const bool scratch = lq_lora_share_bytes(p->M, p->N, p->out_dtype) > 0;
  if (scratch && !q->share) return fail(LQ_ERR_NULL, "lora_linear: share must be non-null for 16-bit outputs of %d tokens", p->M);
  if (scratch && (reinterpret_cast<uintptr_t>(q->share) & 15u)) return fail(LQ_ERR_ALIGN, "lora_linear: share starts on a 16-byte boundary");
  const lora::Shrink s{p->M, p->K, q->L, q->R, RP, 1, values ? stride : p->x_stride, values ? values : p->x, q->a, values ? nullptr : p->x_scale,
                       q->adapters, q->scaling, q->scale, p->M > kFewTokens && p->out_dtype != LQ_F32, q->t};
  Alignment a;
  a.at(q->a).pitch(p->K, size);
  Alignment x;
  if (values) x.at(values).pitch(stride, dtype_bytes(dtype)).pitch(p->K, dtype_bytes(dtype));
  // eight values are one or two accesses of 16 bytes and never leave their row (codes: one of 8, their rows start on 16)
  const bool vec = a.bytes() == 16 && (size == 2 || p->K % 8 == 0) && (values ? x.bytes() == 16 && p->K % 8 == 0 : true);
  // Codes first: the kernel that makes t lets its successors start, which read them ahead of its end
  const bool rows = values && !linear_makes_codes(p);
  if (rows)
    if (int e = lq_quantize_rows(values, dtype, p->M, p->K, stride, const_cast<int8_t*>(p->x), p->x_stride, const_cast<float*>(p->x_scale), stream)) return e;
  const int e = with_dtype(q->dtype, "lora_linear", [&](auto ta) {
    using TA = decltype(ta);
    if (!values) return lora::run_shrink<int8_t, TA>(s, vec, st);
    return with_dtype(dtype, "lora_linear", [&](auto tx) { return lora::run_shrink<decltype(tx), TA>(s, vec, st); });
  });
  if (e != LQ_OK) return e;
  Lora add{q->L, q->R, RP, q->dtype, q->b, q->adapters, q->t, nullptr, 0};
  if (p->M <= kFewTokens) return values && !rows ? run_linear_values(p, &add, values, dtype, stride, st) : run_linear(p, &add, st);
  if (!scratch) {
    add.share = reinterpret_cast<float*>(p->y);
    if (int e2 = lora::expand(add, p, st)) return e2;
    return run_linear(p, &add, st);
  }
  const lora::Slabs slabs(p->M, p->N);
  add.share = q->share;
  add.blocks = (int)slabs.blocks;
  for (long long i = 0; i < slabs.count; ++i) {
    const int from = slabs.start(i);
    lq_linear_problem part = *p;
    part.M = slabs.start(i + 1) - from;
    part.x = p->x + from * p->x_stride;
    part.x_scale = p->x_scale + from;
    part.y = reinterpret_cast<uint16_t*>(p->y) + (size_t)from * p->N;
    add.adapters = q->adapters + from;
    add.t = q->t + (size_t)from * RP;
    if (int e2 = lora::expand(add, &part, st)) return e2;
    if (int e2 = run_linear(&part, &add, st)) return e2;
  }
  return LQ_OK;
}
