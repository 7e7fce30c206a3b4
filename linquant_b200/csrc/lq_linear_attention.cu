// Linear attention with a decay for each head, in floating point.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t                     S [K,V] a head, fp32
//
// Prompts, by chunks of C tokens: with G the running sum of g inside a chunk and S the state that enters it
//   o_i = scale (exp(G_i) q_i S + sum_{j<=i} exp(G_i - G_j) (q_i . k_j) v_j),   S' = exp(G_C) S + sum_j exp(G_C - G_j) k_j v_j^T
// so a chunk is four matrix products. A CTA has VT value channels of one head, keeps its part of the state in the
// accumulators of the last product and walks over the chunks: the data are read once, and nothing but o is written.
// Where a batch has too few heads for the GPU, the tokens are cut into segments: a first pass leaves every segment's own
// state, a small kernel carries them on, and the second pass starts each segment from what enters it.
//
// Rounding. G is summed and kept as two floats, so that differences of large sums are exact; decays are 2^x of fp32
// differences. Products of 16-bit values are exact and their sums fp32. The decayed keys of the state's product are fp32 and go in
// as three bf16 pieces (all 24 bits; fp16: two pieces under a power of two of the largest of them, 22 bits), the state that q
// reads and the decayed products q.k as two pieces (16 or 22 bits). fp32 operands are three bf16 pieces each, six products.
//
// 16-bit prompts whose rows TMA takes run in lq_linear_attention_tc.cu (4 x 4096 x 16 heads of 128 x 128, bf16: 102 us, 334 here, 600 with heads off 16-byte
// boundaries, whose values come one by one; of 256 x 128 968, fp32 957). What is left is bound by warp MMA's own latencies: 5 x 611 x 6 heads of 72 x 100, fp32, 87 us with the call, tensor pipe 29 % busy, HBM 1 %.
#include <math_constants.h>

#include "lq_linear_attention.cuh"

namespace lq {

namespace attention {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// bytes behind the first `bytes` are zero
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// A tile of 16-bit rows of ROWB bytes: 16-byte pieces exclusive-or the row's number, so that eight rows of a piece lie on banks of their own
template <int ROWB>
__device__ __forceinline__ uint32_t at(int row, int piece) {
  return row * ROWB + ((piece ^ (ROWB >= 128 ? row & 7 : (row >> 1) & 3)) << 4);
}

template <typename M>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<M, __half>) mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
  else mma_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
}
// KP: channels of q and k, padded; VT: value channels of the CTA; C: tokens of a chunk
template <typename T, int KP, int VT, int C>
struct Shape {
  using M = typename Half<T>::type;
  static constexpr bool F16 = std::is_same_v<T, __half>;
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;        // pieces of q, k, v
  static constexpr int NK = F16 ? 2 : 3, NS = sizeof(T) == 4 ? 3 : 2, NA = NS;  // pieces of decayed keys, of the state, of decayed q.k
  static constexpr int BUFS = NP == 1 ? 2 : 1;
  static constexpr int QK = C * KP * 2, VB = C * VT * 2, SB = KP * VT * 2;
  static constexpr int TILES = NP * (2 * QK + VB);         // a buffer: q, k, v
  static constexpr int GB = Decay<C>::BYTES;
  static constexpr int ST = BUFS * TILES, GO = ST + NS * SB, RED = GO + GB;
  static constexpr size_t SMEM = RED + 16;
  // Warps: fp32 operands to 128 channels, whose tiles leave room for one CTA an SM, take eight (611 tokens of 6 heads, 72 x 100: one warp a scheduler
  // waits for its own results five clocks of six)
  static constexpr int WARPS = sizeof(T) == 4 && KP <= 128 ? 8 : 4, THREADS = 32 * WARPS;
  static constexpr int WPM = 16 * WARPS / C;               // warps that share 16 rows of the output
  static constexpr int ROWS = WARPS < KP / 16 ? WARPS : KP / 16;  // warps along the state's rows; the others along its columns
  static constexpr int MT = KP / 16 / ROWS, NT = VT / 8 / (WARPS / ROWS);  // a warp's tiles of the state
  static constexpr int REGS = MT * NT * 4;                 // of the state, a thread
};

// Rows of a chunk to a tile: 16-bit values as they are, fp32 as three tiles of bf16 pieces. `vec`: bytes of an access that every row start allows.
template <typename T, int COLS, int C, int PIECE, int NTHREADS>
__device__ __forceinline__ void load_tile(uint32_t dst, const T* src, long long stride, int rows, int cols, int vec) {
  constexpr int ROWB = COLS * 2, PER = COLS / 8;
  if constexpr (sizeof(T) == 2) {
    if (vec == 16) {
#pragma unroll 4
      for (int i = threadIdx.x; i < C * PER; i += NTHREADS) {
        const int row = i / PER, p = i % PER, bytes = row < rows ? min(max(cols - p * 8, 0) * 2, 16) : 0;
        cp_async16_zfill(dst + at<ROWB>(row, p), bytes ? src + row * stride + p * 8 : src, bytes);
      }
    } else if (vec >= 4) {
#pragma unroll 4
      for (int i = threadIdx.x; i < C * PER * 4; i += NTHREADS) {
        const int row = i / (PER * 4), e = i % (PER * 4), bytes = row < rows ? min(max(cols - e * 2, 0) * 2, 4) : 0;
        cp_async4_zfill(dst + at<ROWB>(row, e >> 2) + (e & 3) * 4, bytes ? src + row * stride + e * 2 : src, bytes);
      }
    } else {
#pragma unroll 4
      for (int i = threadIdx.x; i < C * COLS; i += NTHREADS) {
        const int row = i / COLS, e = i % COLS;
        uint16_t v = 0;
        if (row < rows && e < cols) v = __ldg(reinterpret_cast<const unsigned short*>(src) + row * stride + e);
        sts_u16(dst + at<ROWB>(row, e >> 3) + (e & 7) * 2, v);
      }
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < C * PER; i += NTHREADS) {
      const int row = i / PER, p = i % PER;
      const float* from = src + row * stride + p * 8;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        if (vec == 16 && row < rows && p * 8 + e + 4 <= cols) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(from + e));
          x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[e + j] = row < rows && p * 8 + e + j < cols ? __ldg(from + e + j) : 0.f;
        }
      }
      uint32_t hi[4], mid[4], lo[4];
      split3(x, hi, mid, lo);
      const uint32_t to = dst + at<ROWB>(row, p);
      sts_v4(to, hi);
      sts_v4(to + PIECE, mid);
      sts_v4(to + 2 * PIECE, lo);
    }
  }
}

// A chunk's rows on their way to L2
template <int NTHREADS>
__device__ __forceinline__ void prefetch_tile(const float* src, long long stride, int rows, int cols) {
  const int lines = (cols + 31) / 32;
  for (int i = threadIdx.x; i < rows * lines; i += NTHREADS)
    asm volatile("prefetch.global.L2 [%0];\n" ::"l"(src + i / lines * stride + i % lines * 32));
}

struct Vec {
  int q, k, v, o;  // bytes of an access
};

template <typename T, int KP, int VT, int C, bool STATES>
__global__ void __launch_bounds__(sizeof(T) == 4 && KP <= 128 ? 256 : 128, sizeof(T) == 2 && KP <= 128 ? 2 : 1) linear_attention_kernel(const lq_attention_problem p, const Segments seg, const Vec vec) {
  using S = Shape<T, KP, VT, C>;
  using M = typename S::M;
  constexpr bool F16 = S::F16;
  constexpr int NP = S::NP, MT = S::MT, NT = S::NT, KS = KP / 16, CS = C / 16;
  constexpr int SIDE = 2;  // pairs of sums side by side: a sum's products wait for one another
  // fp32 operands: the six products of a step sum by themselves and join the others by an addition that rounds. The tensor core cuts
  // its sums off, always towards zero: over the 72 products of an output or those of all tokens of a state that adds up to 1e-6.
  constexpr bool APART = NP == 3;
  float own[APART ? SIDE : 1][2][4];
  auto sum = [&](float (&all)[4], int u, int half) -> float(&)[4] {
    if constexpr (APART) return own[u][half];
    else return all;
  };
  auto start = [&]() {
    if constexpr (APART)
#pragma unroll
      for (int u = 0; u < SIDE; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) own[u][e >> 2][e & 3] = 0.f;
  };
  auto join = [&](float (&all)[4], int u, int half) {
    if constexpr (APART)
#pragma unroll
      for (int e = 0; e < 4; ++e) all[e] += own[u][half][e];
  };
  extern __shared__ __align__(128) uint8_t smem_dyn[];
  const uint32_t s0 = smem_u32(smem_dyn), s_state = s0 + S::ST, s_red = s0 + S::RED;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int vts = (p.V + VT - 1) / VT, bh = blockIdx.x / vts, vt = blockIdx.x % vts, b = bh / p.H, h = bh % p.H, v0 = vt * VT;
  const int hk = h / (p.H / p.Hk);
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = blockIdx.y * seg.tokens, last_token = (int)min((long long)first + seg.tokens, (long long)p.T), stop = min(n, last_token);
  const int chunks = stop > first ? (stop - first + C - 1) / C : 0;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + hk * p.q_stride_h;
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_stride_b + hk * p.k_stride_h;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_stride_b + h * p.v_stride_h + v0;
  const int cols = min(VT, p.V - v0);

  float st[MT][NT][4];  // rows d0 + 16 m + g (+ 8), columns 8 (js + j) + 2 t4 (+ 1); fp16: times 2^-exp_w
  const int d0 = warp % S::ROWS * (16 * MT), js = warp / S::ROWS * NT;
  int exp_w = 0;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[m][j][e] = 0.f;
  const size_t tile = (size_t)blockIdx.x * S::THREADS * S::REGS;
  if (blockIdx.y > 0) {
    if constexpr (!STATES) {
      const float4* from = reinterpret_cast<const float4*>(seg.states + (size_t)(blockIdx.y - 1) * gridDim.x * S::THREADS * S::REGS + tile);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float4 x = from[(m * NT + j) * S::THREADS + tid];
          st[m][j][0] = x.x, st[m][j][1] = x.y, st[m][j][2] = x.z, st[m][j][3] = x.w;
        }
    }
  } else if (p.initial_state != nullptr) {
    const float* from = p.initial_state + (size_t)bh * p.K * p.V + v0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = d0 + 16 * m + g + 8 * (e >> 1), c = 8 * (js + j) + 2 * t4 + (e & 1);
          if (d < p.K && c < cols) st[m][j][e] = __ldg(from + (size_t)d * p.V + c);
        }
  }

  auto load = [&](int c, int buf) {
    const int t0 = first + c * C, rows = min(C, stop - t0);
    const uint32_t to = s0 + buf * S::TILES;
    if constexpr (!STATES) load_tile<T, KP, C, S::QK, S::THREADS>(to, q + t0 * p.q_stride_t, p.q_stride_t, rows, p.K, vec.q);
    load_tile<T, KP, C, S::QK, S::THREADS>(to + NP * S::QK, k + t0 * p.k_stride_t, p.k_stride_t, rows, p.K, vec.k);
    load_tile<T, VT, C, S::VB, S::THREADS>(to + 2 * NP * S::QK, v + t0 * p.v_stride_t, p.v_stride_t, rows, cols, vec.v);
    cp_async_commit();
  };
  // what q reads: the state in pieces; fp16: under a power of two that all warps share
  int exp_c = 0;
  auto largest = [&]() {
    float top = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fabsf(st[m][j][e]) < CUDART_INF_F ? fmaxf(top, fabsf(st[m][j][e])) : top;  // an infinity scales nothing
#pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    if (lane == 0) sts_u32(s_red + 4 * warp, __float_as_uint(top * pow2(exp_w)));
  };
  auto publish = [&]() {
    float f = 1.f;
    if constexpr (F16) {
      exp_c = exponent(fmaxf(fmaxf(lds_f32(s_red), lds_f32(s_red + 4)), fmaxf(lds_f32(s_red + 8), lds_f32(s_red + 12)))) - 14;
      f = pow2(exp_w - exp_c);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int d = d0 + 16 * m + g + 8 * r;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t w[S::NS];
          split<M, S::NS>(st[m][j][2 * r] * f, st[m][j][2 * r + 1] * f, w);
          const uint32_t to = s_state + at<VT * 2>(d, js + j) + 4 * t4;
#pragma unroll
          for (int i = 0; i < S::NS; ++i) sts_u32(to + i * S::SB, w[i]);
        }
      }
  };

  const uint32_t s_g = s0 + S::GO;
  Pair total;  // warp 0: the segment's log-decay
  Decay<C> next;
  float x_next[C / 32];
  if (chunks > 0) {
    load(0, 0);
    if (warp == 0) {
      load_decay<C>(x_next, p, b, h, first, stop);
      total = next.of(x_next);
      next.store(s_g);
      load_decay<C>(x_next, p, b, h, first + C, stop);
    }
    if constexpr (!STATES) {
      if constexpr (F16) {
        largest();
        __syncthreads();
      }
      publish();
    }
  }
  for (int c = 0; c < chunks; ++c) {
    const int buf = S::BUFS == 2 ? c & 1 : 0, t0 = first + c * C;
    const uint32_t s_q = s0 + buf * S::TILES, s_k = s_q + NP * S::QK, s_v = s_k + NP * S::QK;
    cp_async_wait<0>();
    __syncthreads();  // tiles, decays and the state's pieces are there
    if (S::BUFS == 2 && c + 1 < chunks) load(c + 1, buf ^ 1);
    if constexpr (sizeof(T) == 4) {
      const int t1 = t0 + C, rows = min(C, stop - t1);
      if (!STATES) prefetch_tile<S::THREADS>(q + t1 * p.q_stride_t, p.q_stride_t, rows, p.K);
      prefetch_tile<S::THREADS>(k + t1 * p.k_stride_t, p.k_stride_t, rows, p.K);
      prefetch_tile<S::THREADS>(v + t1 * p.v_stride_t, p.v_stride_t, rows, cols);
    }
    if (warp == 0 && c + 1 < chunks) {
      total = total + next.of(x_next);
      load_decay<C>(x_next, p, b, h, t0 + 2 * C, stop);
    }
    if constexpr (!STATES) {
      const int mt = warp / S::WPM, r0 = 16 * mt;  // rows of this warp; of the VT columns it has its share
      constexpr int NV = VT / 8 / S::WPM, SV = NV >= 4 ? SIDE : 1;
      const int j0 = warp % S::WPM * NV;
      // decayed products of q and k
      float a[2 * CS][4];
#pragma unroll
      for (int j = 0; j < 2 * CS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[j][e] = 0.f;
      const int arow = r0 + (lane & 15), apiece = lane >> 4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (16 * ks >= p.K) break;
        uint32_t qa[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i) ldsm4(qa[i], s_q + i * S::QK + at<KP * 2>(arow, 2 * ks + apiece));
#pragma unroll
        for (int j = 0; j < CS; j += SIDE) {
          if (j > mt) break;
          start();
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t kb[SIDE][4];
#pragma unroll
            for (int u = 0; u < SIDE; ++u) ldsm4(kb[u], s_k + i * S::QK + at<KP * 2>(16 * (j + u) + (lane & 7) + (lane >> 4) * 8, 2 * ks + ((lane >> 3) & 1)));
#pragma unroll
            for (int o = NP - 1 - i; o >= 0; --o)
#pragma unroll
              for (int u = 0; u < SIDE; ++u) {
                if (j + u > mt) break;
                mma<M>(sum(a[2 * (j + u)], u, 0), qa[o], kb[u][0], kb[u][1]);
                mma<M>(sum(a[2 * (j + u) + 1], u, 1), qa[o], kb[u][2], kb[u][3]);
              }
          }
#pragma unroll
          for (int u = 0; u < SIDE; ++u) join(a[2 * (j + u)], u, 0), join(a[2 * (j + u) + 1], u, 1);
        }
      }
      decay_products<C>(a, s_g, r0, 2 * mt + 2);
      float up0 = 1.f, up1 = 1.f;
      if constexpr (F16) row_scales(a, 2 * mt + 2, up0, up1);
      uint32_t pa[S::NA][CS][4];
#pragma unroll
      for (int j = 0; j < CS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int jj = 2 * j + (e >> 1), r = (e & 1) * 2;
          const float up = F16 ? (e & 1 ? up1 : up0) : 1.f;
          uint32_t w[S::NA];
          split<M, S::NA>(F16 ? a[jj][r] * up : a[jj][r], F16 ? a[jj][r + 1] * up : a[jj][r + 1], w);
#pragma unroll
          for (int i = 0; i < S::NA; ++i) pa[i][j][e] = w[i];
        }
      // q S
      float o[NV][4];
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (16 * ks >= p.K) break;
        uint32_t qa[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i) ldsm4(qa[i], s_q + i * S::QK + at<KP * 2>(arow, 2 * ks + apiece));
#pragma unroll
        for (int j = 0; j < NV; j += 2 * SV) {
          start();
#pragma unroll
          for (int i = S::NS - 1; i >= 0; --i) {
            uint32_t sb[SV][4];
#pragma unroll
            for (int u = 0; u < SV; ++u) ldsm4t(sb[u], s_state + i * S::SB + at<VT * 2>(16 * ks + (lane & 15), j0 + j + 2 * u + (lane >> 4)));
#pragma unroll
            for (int w = NP - 1; w >= 0; --w) {
              if (w + i >= S::NS) continue;
#pragma unroll
              for (int u = 0; u < SV; ++u) {
                mma<M>(sum(o[j + 2 * u], u, 0), qa[w], sb[u][0], sb[u][1]);
                mma<M>(sum(o[j + 2 * u + 1], u, 1), qa[w], sb[u][2], sb[u][3]);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < SV; ++u) join(o[j + 2 * u], u, 0), join(o[j + 2 * u + 1], u, 1);
        }
      }
      const float f0 = ex2(lds_f32(s_g + 4 * (r0 + g))) * (F16 ? pow2(exp_c) : 1.f) * up0;
      const float f1 = ex2(lds_f32(s_g + 4 * (r0 + g + 8))) * (F16 ? pow2(exp_c) : 1.f) * up1;
#pragma unroll
      for (int j = 0; j < NV; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
      // and the chunk's own tokens
#pragma unroll
      for (int ks = 0; ks < CS; ++ks) {
        if (ks > mt) break;
#pragma unroll
        for (int j = 0; j < NV; j += 2 * SV) {
          start();
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t vb[SV][4];
#pragma unroll
            for (int u = 0; u < SV; ++u) ldsm4t(vb[u], s_v + i * S::VB + at<VT * 2>(16 * ks + (lane & 15), j0 + j + 2 * u + (lane >> 4)));
#pragma unroll
            for (int w = S::NA - 1 - i; w >= 0; --w)
#pragma unroll
              for (int u = 0; u < SV; ++u) {
                mma<M>(sum(o[j + 2 * u], u, 0), pa[w][ks], vb[u][0], vb[u][1]);
                mma<M>(sum(o[j + 2 * u + 1], u, 1), pa[w][ks], vb[u][2], vb[u][3]);
              }
          }
#pragma unroll
          for (int u = 0; u < SV; ++u) join(o[j + 2 * u], u, 0), join(o[j + 2 * u + 1], u, 1);
        }
      }
      const float c0 = F16 ? p.scale / up0 : p.scale, c1 = F16 ? p.scale / up1 : p.scale;
      const bool in0 = t0 + r0 + g < stop, in1 = t0 + r0 + g + 8 < stop;
      T* out = reinterpret_cast<T*>(p.o) + ((size_t)b * p.T * p.H + h) * p.V + v0;
      const size_t pitch = (size_t)p.H * p.V;
#pragma unroll
      for (int j = 0; j < NV; ++j) {  // rows behind the sequence are zero
        o[j][0] = in0 ? o[j][0] * c0 : 0.f, o[j][1] = in0 ? o[j][1] * c0 : 0.f;
        o[j][2] = in1 ? o[j][2] * c1 : 0.f, o[j][3] = in1 ? o[j][3] * c1 : 0.f;
      }
      if (sizeof(T) == 2 && vec.o == 16) {  // through the warp's own rows of q, which nobody reads any more
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          sts_u32(s_q + at<KP * 2>(r0 + g, j) + 4 * t4, Act<M>::pack2(o[j][0], o[j][1]));
          sts_u32(s_q + at<KP * 2>(r0 + g + 8, j) + 4 * t4, Act<M>::pack2(o[j][2], o[j][3]));
        }
        __syncwarp();
#pragma unroll
        for (int i = lane; i < 16 * NV; i += 32) {
          const int row = i / NV, piece = i % NV;
          uint32_t w[4];
          lds_v4(s_q + at<KP * 2>(r0 + row, piece), w);
          if (t0 + r0 + row < last_token && piece * 8 < cols)
            *reinterpret_cast<uint4*>(out + (size_t)(t0 + r0 + row) * pitch + piece * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int t = t0 + r0 + g + 8 * r, col = 8 * (j0 + j) + 2 * t4;
            if (t >= last_token) continue;
            T* to = out + (size_t)t * pitch + col;
            if (vec.o >= 2 * (int)sizeof(T) && col + 1 < cols) {
              Pack<T, 2> w;
              const float x[2] = {o[j][2 * r], o[j][2 * r + 1]};
              w.set(x);
              store_pack(to, w);
            } else {
              if (col < cols) to[0] = from_f32<T>(o[j][2 * r]);
              if (col + 1 < cols) to[1] = from_f32<T>(o[j][2 * r + 1]);
            }
          }
      }
    }
    // the state
    {
      uint32_t ka[NP][CS][4];
      const float decay = lds_f32(s_g + 12 * C);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int piece = (d0 + 16 * m) / 8 + ((lane >> 3) & 1);
#pragma unroll
        for (int ks = 0; ks < CS; ++ks)
#pragma unroll
          for (int i = 0; i < NP; ++i) ldsm4t(ka[i][ks], s_k + i * S::QK + at<KP * 2>(16 * ks + (lane & 7) + (lane >> 4) * 8, piece));
        float down = 1.f;
        if constexpr (F16) {
          if (m == 0) {  // a power of two above the warp's largest decayed key, each under its own token's decay
            float big = 0.f;
#pragma unroll
            for (int ks = 0; ks < CS; ++ks) {
              const float2 w0 = lds_f2(s_g + 4 * (2 * C + 16 * ks + 2 * t4)), w1 = lds_f2(s_g + 4 * (2 * C + 16 * ks + 8 + 2 * t4));
              __half2 top[2] = {__half2half2(__ushort_as_half(0)), __half2half2(__ushort_as_half(0))};  // of tokens 2 t4 (+ 1), and of those 8 behind them
#pragma unroll
              for (int mm = 0; mm < MT; ++mm) {
                uint32_t r[4];
                ldsm4t(r, s_k + at<KP * 2>(16 * ks + (lane & 7) + (lane >> 4) * 8, (d0 + 16 * mm) / 8 + ((lane >> 3) & 1)));
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e >> 1] = __hmax2(top[e >> 1], __habs2(*reinterpret_cast<__half2*>(&r[e])));
              }
              big = fmaxf(big, fmaxf(fminf(__low2float(top[0]), 65504.f) * w0.x, fminf(__high2float(top[0]), 65504.f) * w0.y));
              big = fmaxf(big, fmaxf(fminf(__low2float(top[1]), 65504.f) * w1.x, fminf(__high2float(top[1]), 65504.f) * w1.y));
            }
#pragma unroll
            for (int x = 16; x; x >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
            const int to = big > 0.f ? max(min(exponent(big) - 14, 100), -100) : exp_w;
            const float move = pow2(exp_w - to);
#pragma unroll
            for (int mm = 0; mm < MT; ++mm)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) st[mm][j][e] *= move;
            exp_w = to;
          }
          down = pow2(-exp_w);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[m][j][e] *= decay;
#pragma unroll
        for (int ks = 0; ks < CS; ++ks) {
          const float2 w0 = lds_f2(s_g + 4 * (2 * C + 16 * ks + 2 * t4)), w1 = lds_f2(s_g + 4 * (2 * C + 16 * ks + 8 + 2 * t4));
          uint32_t kp[S::NK][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = Act<M>::get(ka[0][ks][e], 0), y = Act<M>::get(ka[0][ks][e], 1);
            if constexpr (NP == 3) {  // the whole value again, exactly
              x += Act<M>::get(ka[1][ks][e], 0) + Act<M>::get(ka[2][ks][e], 0);
              y += Act<M>::get(ka[1][ks][e], 1) + Act<M>::get(ka[2][ks][e], 1);
            }
            const float2 w = e < 2 ? w0 : w1;
            x *= w.x, y *= w.y;
            if constexpr (F16) x *= down, y *= down;
            uint32_t pieces[S::NK];
            split<M, S::NK>(x, y, pieces);
#pragma unroll
            for (int i = 0; i < S::NK; ++i) kp[i][e] = pieces[i];
          }
#pragma unroll
          for (int j = 0; j < NT; j += 2 * SIDE) {
            start();
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              uint32_t vb[SIDE][4];
#pragma unroll
              for (int u = 0; u < SIDE; ++u) ldsm4t(vb[u], s_v + i * S::VB + at<VT * 2>(16 * ks + (lane & 15), js + j + 2 * u + (lane >> 4)));
#pragma unroll
              for (int w = S::NK - 1 - i; w >= 0; --w)
#pragma unroll
                for (int u = 0; u < SIDE; ++u) {
                  mma<M>(sum(st[m][j + 2 * u], u, 0), kp[w], vb[u][0], vb[u][1]);
                  mma<M>(sum(st[m][j + 2 * u + 1], u, 1), kp[w], vb[u][2], vb[u][3]);
                }
            }
#pragma unroll
            for (int u = 0; u < SIDE; ++u) join(st[m][j + 2 * u], u, 0), join(st[m][j + 2 * u + 1], u, 1);
          }
        }
      }
    }
    if (c + 1 < chunks) {
      if constexpr (!STATES && F16) largest();
      __syncthreads();  // the decays, the state's pieces and the tiles of this chunk have been read
      if (warp == 0) next.store(s_g);
      if constexpr (!STATES) publish();
      if (S::BUFS == 1) load(c + 1, 0);
    }
  }

  const float back = F16 ? pow2(exp_w) : 1.f;
  if constexpr (STATES) {
    float4* to = reinterpret_cast<float4*>(seg.states + (size_t)blockIdx.y * gridDim.x * S::THREADS * S::REGS + tile);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        to[(m * NT + j) * S::THREADS + tid] = make_float4(st[m][j][0] * back, st[m][j][1] * back, st[m][j][2] * back, st[m][j][3] * back);
    if (vt == 0 && tid == 0) seg.decays[(size_t)blockIdx.y * (gridDim.x / vts) + bh] = total.hi;
  } else {
    if (p.final_state != nullptr && (int)blockIdx.y == (n > 0 ? (n - 1) / seg.tokens : 0)) {
      float* to = p.final_state + (size_t)bh * p.K * p.V + v0;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = d0 + 16 * m + g + 8 * (e >> 1), col = 8 * (js + j) + 2 * t4 + (e & 1);
            if (d < p.K && col < cols) to[(size_t)d * p.V + col] = st[m][j][e] * back;
          }
    }
    // tokens behind the sequence, from the first whole chunk that has none of it
    T* out = reinterpret_cast<T*>(p.o) + ((size_t)b * p.T * p.H + h) * p.V + v0;
    const int from = first + chunks * C;
    for (long long i = tid; i < (long long)max(last_token - from, 0) * VT; i += S::THREADS) {
      const int col = (int)(i % VT);
      if (col < cols) out[(size_t)(from + i / VT) * p.H * p.V + col] = from_f32<T>(0.f);
    }
  }
}

// What leaves a segment: its own state and, decayed, what entered it. One thread has four values of all segments, eight of them on their way.
// The decay goes in by its square root, twice: tokens that grow may multiply a segment by more than fp32 holds where what they multiply is small, or zero.
__global__ void __launch_bounds__(128) segment_states_kernel(const Segments seg, int heads, long long values, int values_a_head) {
  constexpr int U = 8;
  pdl_enter();
  const long long i = (blockIdx.x * 128ll + threadIdx.x) * 4;
  if (i >= values) return;
  const int bh = (int)(i / values_a_head), last = seg.count - 2;  // the last segment's is not there
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 <= last; k0 += U) {
    float4 own[U];
    float a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(k0 + u, last);
      own[u] = *reinterpret_cast<const float4*>(seg.states + (size_t)k * values + i);
      a[u] = ex2(0.5f * __ldg(seg.decays + (size_t)k * heads + bh));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u;
      if (k > last) break;
      auto on = [&](float before, float own) { return before == 0.f ? own : fmaf(a[u], a[u] * before, own); };
      s = k == 0 ? own[u] : make_float4(on(s.x, own[u].x), on(s.y, own[u].y), on(s.z, own[u].z), on(s.w, own[u].w));
      if (k > 0) *reinterpret_cast<float4*>(seg.states + (size_t)k * values + i) = s;
    }
  }
}

// ---- single tokens: the state is read and written once. A row of V values is LPR lanes wide, warps share the K rows; four rows of 16
// bytes a thread are on their way. Bound by the state's bytes: 128 sequences of 16 heads, 128 x 128 fp32, 51 us, 5.2 TB/s; one: 2.1 us.
template <typename T, typename TS, int VW, int LPR>
__global__ void __launch_bounds__(256) linear_attention_step_kernel(const lq_attention_problem p) {
  constexpr int ROWS = 256 / LPR, U = 4;  // rows of a round, rounds in flight
  __shared__ float part[8][LPR * VW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, col = (blockIdx.x * LPR + tid % LPR) * VW, row0 = tid / LPR;
  const int h = blockIdx.y, hk = h / (p.H / p.Hk);
  pdl_enter();
  for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
    T* o = reinterpret_cast<T*>(p.o) + ((size_t)b * p.H + h) * p.V + col;
    const int slot = p.slots ? __ldg(p.slots + b) : b;
    if (slot < 0 || slot >= p.n_slots) {  // an idle entry
      if (tid < LPR)
        for (int i = 0; i < VW; ++i)
          if (col + i < p.V) o[i] = from_f32<T>(0.f);
      continue;
    }
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + hk * p.q_stride_h;
    const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_stride_b + hk * p.k_stride_h;
    const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_stride_b + h * p.v_stride_h;
    TS* s = reinterpret_cast<TS*>(p.state) + ((size_t)slot * p.H + h) * p.K * p.V + col;
    const float a = p.g ? expf(__ldg(p.g + b * p.g_stride_b + h * p.g_stride_h)) : 1.f;
    const bool on = col < p.V;
    float vv[VW], sum[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) vv[i] = col + i < p.V ? to_f32(v[col + i]) : 0.f, sum[i] = 0.f;
    for (int d0 = row0; d0 < p.K; d0 += ROWS * U) {
      Pack<TS, VW> raw[U];
      float kd[U], qd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int d = d0 + u * ROWS;
        const bool in = on && d < p.K;
        raw[u].zero();
        if (in) raw[u] = load_pack<TS, VW>(s + (size_t)d * p.V);
        kd[u] = in ? to_f32(k[d]) : 0.f;
        qd[u] = in ? to_f32(q[d]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int d = d0 + u * ROWS;
        float x[VW];
        raw[u].get(x);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          x[i] = fmaf(a, x[i], kd[u] * vv[i]);
          sum[i] = fmaf(qd[u], x[i], sum[i]);
        }
        raw[u].set(x);
        if (on && d < p.K) store_pack(s + (size_t)d * p.V, raw[u]);
      }
    }
#pragma unroll
    for (int m = LPR; m < 32; m <<= 1)
#pragma unroll
      for (int i = 0; i < VW; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], m);
    if (lane < LPR)
#pragma unroll
      for (int i = 0; i < VW; ++i) part[warp][lane * VW + i] = sum[i];
    __syncthreads();
    for (int c = tid; c < LPR * VW; c += 256) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) x += part[w][c];
      const int at = blockIdx.x * LPR * VW + c;
      if (at < p.V) reinterpret_cast<T*>(p.o)[((size_t)b * p.H + h) * p.V + at] = from_f32<T>(x * p.scale);
    }
    __syncthreads();
  }
}

cudaError_t launch_segment_states(const Segments& seg, int heads, long long values, cudaStream_t st) {
  return launch(segment_states_kernel, dim3((unsigned)((values / 4 + 127) / 128)), dim3(128), 0, st, seg, heads, values, (int)(values / heads));
}

static int check(const lq_attention_problem* p, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->B < 0 || p->T < 0 || p->H <= 0 || p->Hk <= 0 || p->H % p->Hk || p->K <= 0 || p->V <= 0 || !fits(p->B) || !fits(p->T) || !fits(p->V))
    return fail(LQ_ERR_SHAPE, "%s: B=%d T=%d H=%d Hk=%d K=%d V=%d", what, p->B, p->T, p->H, p->Hk, p->K, p->V);
  if (p->K > 256) return fail(LQ_ERR_UNSUPPORTED, "%s: K=%d, at most 256 channels of q and k", what, p->K);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d", what, p->dtype);
  if ((long long)p->B * p->H * ((p->V + 31) / 32) >= 1ll << 30) return fail(LQ_ERR_SHAPE, "%s: B=%d H=%d V=%d", what, p->B, p->H, p->V);
  return LQ_OK;
}

// Segments: enough CTAs for every place on the GPU (two an SM, one of fp32 operands or for the tcgen05 kernel). None is shorter than four
// chunks, two of fp32 operands, whose chunks take ten times as long, and calls of fewer than twelve stay whole. 16 heads of 128 x 128, bf16: 512
// tokens whole 12.4 us, in two 14.7; 1024 whole 21.3, in four 17.3; 4 heads, 2048: in four 22.4, in eight 16.3. fp32, 6 heads of
// 72 x 100, 611 tokens: whole 155, in two 113
static Plan plan(const lq_attention_problem* p) {
  Plan r;
  r.tc = tc_applies(p);
  const int kp = p->K <= 64 && !r.tc ? 64 : p->K <= 128 ? 128 : 256, vt = kp == 256 ? 32 : 64;
  r.floats = kp * vt;
  r.tiles = (long long)p->B * p->H * ((p->V + vt - 1) / vt);
  const long long chunks = ((long long)p->T + 63) / 64, room = (r.tc || p->dtype == LQ_F32 ? 1ll : 2ll) * sm_count(), least = p->dtype == LQ_F32 ? 2 : chunks < 12 ? 12 : 4;
  long long count = r.tiles > 0 ? room / r.tiles : 1;
  count = count > chunks / least ? chunks / least : count;
  count = count < 1 ? 1 : count;
  const long long each = (chunks + count - 1) / count;
  r.tokens = (int)((each < 1 ? 1 : each) * 64);
  r.count = (int)((p->T + (long long)r.tokens - 1) / r.tokens);
  if (r.count < 1) r.count = 1;
  return r;
}
static size_t workspace(const lq_attention_problem* p, const Plan& r) {
  if (r.count < 2) return 0;
  return (size_t)(r.count - 1) * ((size_t)r.tiles * r.floats + (((size_t)p->B * p->H + 63) / 64) * 64) * 4;
}

static int access_bytes(const void* ptr, long long sb, long long st, long long sh, int size) {
  Alignment a;
  return a.at(ptr).pitch(sb, size).pitch(st, size).pitch(sh, size).bytes();
}

template <typename T, int KP, int VT, int C>
static int run(const lq_attention_problem* p, const Plan& r, const Segments& seg, cudaStream_t st) {
  using S = Shape<T, KP, VT, C>;
  const int size = sizeof(T);
  const Vec vec{access_bytes(p->q, p->q_stride_b, p->q_stride_t, p->q_stride_h, size), access_bytes(p->k, p->k_stride_b, p->k_stride_t, p->k_stride_h, size),
                access_bytes(p->v, p->v_stride_b, p->v_stride_t, p->v_stride_h, size), access_bytes(p->o, p->V, p->V, p->V, size)};
  const dim3 block(S::THREADS);
  cudaError_t e = cudaSuccess;
  if (seg.count > 1) {
    e = launch_opt_in(linear_attention_kernel<T, KP, VT, C, true>, dim3((unsigned)r.tiles, seg.count - 1), block, S::SMEM, st, *p, seg, vec);
    if (e == cudaSuccess && seg.count > 2) e = launch_segment_states(seg, p->B * p->H, r.tiles * S::THREADS * S::REGS, st);
  }
  if (e == cudaSuccess) e = launch_opt_in(linear_attention_kernel<T, KP, VT, C, false>, dim3((unsigned)r.tiles, seg.count), block, S::SMEM, st, *p, seg, vec);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "linear_attention: %s", cudaGetErrorString(e));
  return check_launch("linear_attention_kernel");
}

}  // namespace attention

}  // namespace lq

extern "C" size_t lq_linear_attention_workspace_bytes(const lq_attention_problem* p) {
  using namespace lq::attention;
  if (check(p, "linear_attention") != LQ_OK || p->B == 0) return 0;
  return workspace(p, plan(p));
}

extern "C" int lq_linear_attention_fwd(const lq_attention_problem* p, void* ws, size_t bytes, lq_stream stream) {
  using namespace lq;
  using namespace lq::attention;
  if (int e = check(p, "linear_attention")) return e;
  if (p->B == 0) return LQ_OK;
  if (p->T > 0 && (!p->q || !p->k || !p->v || !p->o)) return fail(LQ_ERR_NULL, "linear_attention: q, k, v and o must be non-null");
  const Plan r = plan(p);
  const size_t need = workspace(p, r);
  if (need > 0 && (ws == nullptr || bytes < need)) return fail(LQ_ERR_WORKSPACE, "linear_attention: workspace of %zu bytes, %zu needed", bytes, need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 15u)) return fail(LQ_ERR_ALIGN, "linear_attention: workspace must start on a 16-byte boundary");
  float* states = reinterpret_cast<float*>(ws);
  const Segments seg{r.count, r.tokens, states, states + (size_t)(r.count - 1) * r.tiles * r.floats};
  cudaStream_t st = (cudaStream_t)stream;
  if (r.tc) return run_tc(p, r, seg, st);
  return with_dtype(p->dtype, "linear_attention", [&](auto t) {
    using T = decltype(t);
    if (p->K <= 64) return run<T, 64, 64, 64>(p, r, seg, st);
    if (p->K <= 128) return run<T, 128, 64, 64>(p, r, seg, st);
    return run<T, 256, 32, sizeof(T) == 4 ? 32 : 64>(p, r, seg, st);
  });
}

extern "C" int lq_linear_attention_step(const lq_attention_problem* p, lq_stream stream) {
  using namespace lq;
  using namespace lq::attention;
  if (int e = check(p, "linear_attention_step")) return e;
  if (p->T != 1) return fail(LQ_ERR_SHAPE, "linear_attention_step: T=%d, one token", p->T);
  if (p->state_dtype < LQ_F16 || p->state_dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "linear_attention_step: state dtype %d", p->state_dtype);
  if (p->n_slots < 0 || (!p->slots && p->n_slots < p->B)) return fail(LQ_ERR_SHAPE, "linear_attention_step: %d slots for B=%d", p->n_slots, p->B);
  if (p->B == 0) return LQ_OK;
  if (!p->q || !p->k || !p->v || !p->o || (!p->state && p->n_slots > 0)) return fail(LQ_ERR_NULL, "linear_attention_step: q, k, v, o and state must be non-null");
  if (p->H > 65535) return fail(LQ_ERR_SHAPE, "linear_attention_step: H=%d", p->H);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 block(256);
  return with_dtype(p->dtype, "linear_attention_step", [&](auto t) {
    using T = decltype(t);
    return with_dtype(p->state_dtype, "linear_attention_step", [&](auto ts) {
      using TS = decltype(ts);
      constexpr int FULL = 16 / sizeof(TS);
      Alignment a;
      const int bytes = a.at(p->state).pitch(p->V, sizeof(TS)).bytes();
      auto go = [&](auto kern, int tile) {
        const cudaError_t e = launch(kern, dim3((p->V + tile - 1) / tile, p->H, p->B < 65535 ? p->B : 65535), block, 0, st, *p);
        return e != cudaSuccess ? fail(LQ_ERR_LAUNCH, "linear_attention_step: %s", cudaGetErrorString(e)) : check_launch("linear_attention_step_kernel");
      };
      if (bytes == 16) {
        // Few heads: narrow columns, so that more SMs share the states, as long as a round of CTAs takes them (16 heads of 128 x 128, fp32:
        // one sequence 2.1 us, 3.4 with wide ones; 6 sequences 3.1 and 3.6; 8 sequences 4.5 and 3.7)
        if (4ll * p->B * p->H * ((p->V + 32 * FULL - 1) / (32 * FULL)) <= 3ll * sm_count()) return go(linear_attention_step_kernel<T, TS, FULL, 8>, 8 * FULL);
        return go(linear_attention_step_kernel<T, TS, FULL, 32>, 32 * FULL);
      }
      return go(linear_attention_step_kernel<T, TS, 1, 32>, 32);
    });
  });
}
