// Linear attention of prompts on the Blackwell tensor cores: 16-bit operands, K <= 128, rows on 16-byte boundaries.
//
//   o_i = scale (exp(G_i) q_i S + sum_{j<=i} exp(G_i - G_j) (q_i . k_j) v_j),   S' = exp(G_C) S + sum_j k_j (exp(G_C - G_j) v_j)^T
//
// One CTA an SM has 64 value channels of one head and walks over chunks of 64 tokens; its roles run apart by as much as the
// buffers allow, so the only chain from chunk to chunk is the state's own (a few hundred clocks), not the chunk's four products:
//
//   loader warp   q, k, v tiles by TMA into a ring of stages (zeros behind K, V and T), the chunk's decays
//   MMA warp      q k^T; k^T v' (both operands as they lie, token index outermost: "MN-major"); q S; P v
//   warps 0..3    P = decayed q k^T from tensor memory to shared memory, rounded; a chunk later its outputs
//   warps 4..7    v' = exp(G_C - G_j) v in pieces; the state, a row of K a thread in registers, S = a S + k^T v'; S rounded for q
//
// All accumulators lie twice in tensor memory (four of 64 columns). Rounding as in lq_linear_attention.cu with the decay on v instead
// of k (half as many values); here q reads the state as one piece of the type, the same half step as the decayed q k^T has.
// fp16: rows of P, v' of a chunk and the state q reads each under a power of two of their largest value.
// Behind a sequence's last token k and v are made zero in shared memory: a NaN there times a weight of zero would be one.
// Every wait is bounded; on expiry the CTA raises the status word, lets its copies and products land, frees its tensor memory
// and returns.
#include <math_constants.h>

#include "lq_linear_attention.cuh"

namespace lq {

namespace attentiontc {

using namespace attention;

constexpr int C = 64, VT = 64, WARPS = 10, LOADER = 8, ISSUER = 9;
constexpr int TILE = C * 128, QK = 2 * TILE, STAGE = 2 * QK + TILE, STAGES = 3, SB = 128 * 128, GS = 8;  // bytes; GS: chunks whose decays are kept

template <typename T>
struct Shape {
  static constexpr bool F16 = std::is_same_v<T, __half>;
  static constexpr int NV = F16 ? 2 : 3;  // pieces of v'
  static constexpr int VO = STAGES * STAGE, PO = VO + 2 * NV * TILE, SO = PO + 2 * TILE, GO = SO + 2 * SB;
  static constexpr int RED = GO + GS * Decay<C>::BYTES, EXP = RED + 64, BARS = EXP + 16;
  static constexpr int FULL = 0, EMPTY = FULL + STAGES, S1 = EMPTY + STAGES, PF = S1 + 2, VF = PF + 2, DS = VF + 2, SF = DS + 2, OF = SF + 2, OE = OF + 2, LAST = OE + 2, COUNT = LAST + 1;
  static constexpr int TBASE = BARS + 8 * COUNT;
  static constexpr size_t SMEM = 1024 + TBASE + 8;
  static_assert(SMEM <= 232448);
};
// tensor memory: columns of the accumulators
constexpr int T_S1 = 0, T_QS = 128, T_PV = 256, T_DS = 384;

__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity)) != 0; }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
               : "memory");
}
// warps 4..7 decide together
__device__ __forceinline__ bool group_and(bool ok) {
  uint32_t r;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 q, %1, 0;\nbar.red.and.pred p, 1, 128, q;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r) : "r"((uint32_t)ok) : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t place(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
// both operands of one 16-bit type, fp32 sums; MN-major: the reduction index outermost
template <typename T>
__device__ __forceinline__ uint32_t idesc(int M, int N, bool a_mn, bool b_mn) {
  return idesc_f16(M, N) | (std::is_same_v<T, __half> ? 0u : (1u << 7) | (1u << 10)) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}
// MN-major operand of two tiles of 64 that lie `apart` bytes from one another
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr, int apart) {
  return (desc_kmajor_sw128(saddr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(apart >> 4) << 16);
}

template <typename T, bool STATES>
__global__ void __launch_bounds__(32 * WARPS, 1) linear_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                            const __grid_constant__ CUtensorMap map_v, const lq_attention_problem p,
                                                                            const Segments seg, const int wide) {
  using S = Shape<T>;
  constexpr bool F16 = S::F16;
  extern __shared__ __align__(1024) uint8_t smem_dyn[];
  const uint32_t s0 = (smem_u32(smem_dyn) + 1023u) & ~1023u, s_bars = s0 + S::BARS;
  auto bar = [&](int which, int i) { return s_bars + 8u * (which + i); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vts = (p.V + VT - 1) / VT, bh = blockIdx.x / vts, vt = blockIdx.x % vts, b = bh / p.H, h = bh % p.H, v0 = vt * VT;
  const int hk = h / (p.H / p.Hk);
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = blockIdx.y * seg.tokens, last_token = (int)min((long long)first + seg.tokens, (long long)p.T), stop = min(n, last_token);
  const int chunks = stop > first ? (stop - first + C - 1) / C : 0;
  if (tid == 0) {
    for (int i = 0; i < S::COUNT; ++i) {  // PF, VF, SF and OE take an arrival of each of four warps
      const bool four = (i >= S::PF && i < S::DS) || (i >= S::SF && i < S::OF) || (i >= S::OE && i < S::LAST);
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(s_bars + 8u * i), "r"(four ? 4u : 1u));
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(s0 + S::TBASE), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tbase = lds_u32(s0 + S::TBASE);
  bool ok = true;
  auto stage = [&](int c) { return s0 + (uint32_t)(c % STAGES) * STAGE; };
  auto stage_wait = [&](int c) { return warp_wait(bar(S::FULL, c % STAGES), (uint32_t)((c / STAGES) & 1)); };
  auto decays = [&](int c) { return s0 + S::GO + (uint32_t)(c % GS) * Decay<C>::BYTES; };

  if (warp == LOADER) {
    double total = 0;
    float x[C / 32];
    load_decay<C>(x, p, b, h, first, stop);
    Decay<C> d;
    int c = 0;
    for (; c < chunks; ++c) {
      const int s = c % STAGES;
      if (c >= STAGES && !(ok = warp_wait(bar(S::EMPTY, s), (uint32_t)((c / STAGES - 1) & 1)))) break;
      total += d.of(x);
      d.store(decays(c));  // its chunk eight before this one has been left by all: the stages between are empty again
      load_decay<C>(x, p, b, h, first + (c + 1) * C, stop);
      __syncwarp();
      if (lane == 0) {
        const uint32_t to = stage(c), full = bar(S::FULL, s);
        const int t0 = first + c * C;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(full), "r"((uint32_t)(STATES ? QK + TILE : STAGE)) : "memory");
        tma_load_4d(to + QK, &map_k, 0, t0, hk, b, full);
        tma_load_4d(to + QK + TILE, &map_k, 64, t0, hk, b, full);
        if constexpr (!STATES) {
          tma_load_4d(to, &map_q, 0, t0, hk, b, full);
          tma_load_4d(to + TILE, &map_q, 64, t0, hk, b, full);
        }
        tma_load_4d(to + 2 * QK, &map_v, v0, t0, h, b, full);
      }
      __syncwarp();
    }
    for (int k = max(0, c - STAGES); k < c; ++k) ok &= stage_wait(k);  // nothing may land after the CTA has gone
    if (STATES && vt == 0 && lane == 0) seg.decays[(size_t)blockIdx.y * (gridDim.x / vts) + bh] = ex2((float)total);
  } else if (warp == ISSUER) {
    const uint32_t id_s1 = idesc<T>(C, C, false, false), id_mn = idesc<T>(C, VT, false, true), id_ds = idesc<T>(128, VT, true, true);
    auto scores = [&](int c) {
      if (lane == 0) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t at = stage(c) + (ks / 4) * TILE;
          umma_f16(tbase + T_S1 + 64 * (c & 1), desc_kmajor_sw128(at) + 2 * (ks % 4), desc_kmajor_sw128(at + QK) + 2 * (ks % 4), id_s1, ks > 0);
        }
        umma_commit(bar(S::S1, c & 1));
      }
      __syncwarp();
    };
    if constexpr (!STATES) {
      if (chunks > 0 && (ok = stage_wait(0))) {
        after_sync();
        scores(0);
      }
    }
    for (int c = 0; c < chunks && ok; ++c) {
      const int i = c & 1;
      const uint32_t turn = (uint32_t)((c >> 1) & 1);
      if constexpr (!STATES) {
        if (c + 1 < chunks) {  // P of two chunks before has been waited for: its accumulator has been read
          if (!(ok = stage_wait(c + 1))) break;
          after_sync();
          scores(c + 1);
        }
      } else {
        if (c >= 2 && !(ok = warp_wait(bar(S::SF, i), turn ^ 1))) break;
      }
      if (!(ok = warp_wait(bar(S::VF, i), turn))) break;
      after_sync();
      if (lane == 0) {  // the pieces of v', the smallest first
#pragma unroll
        for (int w = S::NV - 1; w >= 0; --w)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_f16(tbase + T_DS + 64 * i, desc_mn_sw128(stage(c) + QK + 2048 * ks, TILE), desc_kmajor_sw128(s0 + S::VO + (i * S::NV + w) * TILE + 2048 * ks), id_ds,
                     w < S::NV - 1 || ks > 0);
        umma_commit(bar(S::DS, i));
        if constexpr (STATES) umma_commit(bar(S::EMPTY, c % STAGES));
      }
      __syncwarp();
      if constexpr (!STATES) {
        if (!(ok = warp_wait(bar(S::SF, i), turn))) break;
        if (c >= 2 && !(ok = warp_wait(bar(S::OE, i), turn ^ 1))) break;
        after_sync();
        if (lane == 0) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks)
            umma_f16(tbase + T_QS + 64 * i, desc_kmajor_sw128(stage(c) + (ks / 4) * TILE) + 2 * (ks % 4), desc_kmajor_sw128(s0 + S::SO + i * SB + 2048 * ks), id_mn, ks > 0);
        }
        __syncwarp();
        if (!(ok = warp_wait(bar(S::PF, i), turn))) break;
        after_sync();
        if (lane == 0) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            umma_f16(tbase + T_PV + 64 * i, desc_kmajor_sw128(s0 + S::PO + i * TILE) + 2 * ks, desc_kmajor_sw128(stage(c) + 2 * QK + 2048 * ks), id_mn, ks > 0);
          umma_commit(bar(S::OF, i));
          umma_commit(bar(S::EMPTY, c % STAGES));
        }
        __syncwarp();
      }
    }
    if (lane == 0) umma_commit(bar(S::LAST, 0));  // every product that was issued
    __syncwarp();
    ok &= warp_wait(bar(S::LAST, 0), 0);
  } else if (warp < 4) {
    if constexpr (!STATES) {
      const int r0 = 16 * warp, g = lane >> 2, t4 = lane & 3, tiles = 2 * warp + 2;
      const uint32_t lanes = (uint32_t)(32 * warp) << 16;  // M = 64: sixteen rows in each quarter of the lanes
      const int cols = min(VT, p.V - v0);
      T* out = reinterpret_cast<T*>(p.o) + ((size_t)b * p.T * p.H + h) * p.V + v0;
      const size_t pitch = (size_t)p.H * p.V;
      float up0 = 1.f, up1 = 1.f;
      auto outputs = [&](int c, float up0, float up1) {
        const int i = c & 1, t0 = first + c * C;
        if (!(ok = warp_wait(bar(S::OF, i), (uint32_t)((c >> 1) & 1)))) return;
        after_sync();
        uint32_t qs[2][16], pv[2][16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          tmem_ld_16x256b_x4(tbase + lanes + T_QS + 64 * i + 32 * k, qs[k]);
          tmem_ld_16x256b_x4(tbase + lanes + T_PV + 64 * i + 32 * k, pv[k]);
        }
        tmem_wait();
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::OE, i));
        const uint32_t s_g = decays(c), s_p = s0 + S::PO + i * TILE;
        float f0 = ex2(lds_f32(s_g + 4 * (r0 + g))) * p.scale, f1 = ex2(lds_f32(s_g + 4 * (r0 + g + 8))) * p.scale, c0 = p.scale, c1 = p.scale;
        if constexpr (F16) {
          const float e = lds_f32(s0 + S::EXP + 4 * (c & 3));
          f0 *= e, f1 *= e, c0 /= up0, c1 /= up1;
        }
        const bool in0 = t0 + r0 + g < stop, in1 = t0 + r0 + g + 8 < stop;  // rows behind the sequence are zero
        float o[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = fmaf(__uint_as_float(qs[j / 4][4 * (j % 4) + e]), e < 2 ? f0 : f1, __uint_as_float(pv[j / 4][4 * (j % 4) + e]) * (e < 2 ? c0 : c1));
            o[j][e] = (e < 2 ? in0 : in1) ? x : 0.f;
          }
        // through the warp's own rows of P, whose product is done
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sts_u32(s_p + place(r0 + g, j) + 4 * t4, Act<T>::pack2(o[j][0], o[j][1]));
          sts_u32(s_p + place(r0 + g + 8, j) + 4 * t4, Act<T>::pack2(o[j][2], o[j][3]));
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = r0 + 4 * k + (lane >> 3), piece = lane & 7, t = t0 + row;
          uint32_t w[4];
          lds_v4(s_p + place(row, piece), w);
          if (t >= last_token || piece * 8 >= cols) continue;
          T* to = out + (size_t)t * pitch + piece * 8;
          if (wide) {
            *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (piece * 8 + e < cols) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
          }
        }
        __syncwarp();  // the rows have been read
      };
      for (int c = 0; c < chunks && ok; ++c) {
        const int i = c & 1;
        if (!(ok = stage_wait(c) && warp_wait(bar(S::S1, i), (uint32_t)((c >> 1) & 1)))) break;
        after_sync();
        uint32_t r[2][16];
#pragma unroll
        for (int k = 0; k < 2; ++k) tmem_ld_16x256b_x4(tbase + lanes + T_S1 + 64 * i + 32 * k, r[k]);
        tmem_wait();
        float a[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[j][e] = j < tiles ? __uint_as_float(r[j / 4][4 * (j % 4) + e]) : 0.f;
        decay_products<C>(a, decays(c), r0, tiles);
        float w0 = 1.f, w1 = 1.f;
        if constexpr (F16) row_scales(a, tiles, w0, w1);
        const uint32_t s_p = s0 + S::PO + i * TILE;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sts_u32(s_p + place(r0 + g, j) + 4 * t4, F16 ? Act<T>::pack2(a[j][0] * w0, a[j][1] * w0) : Act<T>::pack2(a[j][0], a[j][1]));
          sts_u32(s_p + place(r0 + g + 8, j) + 4 * t4, F16 ? Act<T>::pack2(a[j][2] * w1, a[j][3] * w1) : Act<T>::pack2(a[j][2], a[j][3]));
        }
        proxy_fence();
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::PF, i));
        if (c > 0) outputs(c - 1, up0, up1);
        up0 = w0, up1 = w1;
      }
      if (ok && chunks > 0) outputs(chunks - 1, up0, up1);
      // tokens behind the sequence, from the first whole chunk that has none of it
      const int from = first + chunks * C;
      for (long long k = tid; k < (long long)max(last_token - from, 0) * VT; k += 128) {
        const int col = (int)(k % VT);
        if (col < cols) out[(size_t)(from + k / VT) * pitch + col] = from_f32<T>(0.f);
      }
    }
  } else {
    const int d = tid - 128, quad = warp & 3;  // a row of the state, of v' half a token
    const uint32_t lanes = (uint32_t)(32 * quad) << 16;
    const int cols = min(VT, p.V - v0);
    float st[VT];
    const size_t tile = (size_t)blockIdx.x * 128 * VT;
#pragma unroll
    for (int j = 0; j < VT; ++j) st[j] = 0.f;
    if (!STATES && blockIdx.y > 0) {
      const float4* from = reinterpret_cast<const float4*>(seg.states + (size_t)(blockIdx.y - 1) * gridDim.x * 128 * VT + tile);
#pragma unroll
      for (int j = 0; j < VT; j += 4) {
        const float4 x = from[(j / 4) * 128 + d];
        st[j] = x.x, st[j + 1] = x.y, st[j + 2] = x.z, st[j + 3] = x.w;
      }
    } else if (blockIdx.y == 0 && p.initial_state != nullptr && d < p.K) {
      const float* from = p.initial_state + ((size_t)bh * p.K + d) * p.V + v0;
#pragma unroll
      for (int j = 0; j < VT; ++j)
        if (j < cols) st[j] = __ldg(from + j);
    }
    auto group_max = [&](float top, int slot) {  // of warps 4..7, which leave together where a wait ran out
#pragma unroll
      for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
      if (lane == 0) sts_u32(s0 + S::RED + 16 * slot + 4 * quad, __float_as_uint(top));
      ok = group_and(ok);
      const uint32_t at = s0 + S::RED + 16 * slot;
      return fmaxf(fmaxf(lds_f32(at), lds_f32(at + 4)), fmaxf(lds_f32(at + 8), lds_f32(at + 12)));
    };
    auto publish = [&](int c) {
      float f = 1.f;
      if constexpr (F16) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < VT; ++j) top = fabsf(st[j]) < CUDART_INF_F ? fmaxf(top, fabsf(st[j])) : top;  // an infinity scales nothing
        const int e = exponent(group_max(top, 2)) - 14;
        if (!ok) return;
        f = pow2(-e);
        if (d == 0) sts_u32(s0 + S::EXP + 4 * (c & 3), __float_as_uint(pow2(e)));
      }
      const uint32_t to = s0 + S::SO + (c & 1) * SB;
#pragma unroll
      for (int j = 0; j < VT; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = Act<T>::pack2(F16 ? st[j + 2 * e] * f : st[j + 2 * e], F16 ? st[j + 2 * e + 1] * f : st[j + 2 * e + 1]);
        sts_v4(to + place(d, j / 8), w);
      }
      proxy_fence();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S::SF, c & 1));
    };
    float back = 1.f, back_next = 1.f;  // fp16: what the sums of v' are multiplied by
    auto decayed = [&](int c) {
      const int row = d >> 1, half = d & 1, rows = min(C, stop - first - c * C);
      const uint32_t s_k = stage(c) + QK, s_v = stage(c) + 2 * QK, to = s0 + S::VO + (c & 1) * S::NV * TILE;
      if (!(ok &= stage_wait(c)) && !F16) return;
      const float w = lds_f32(decays(c) + 4 * (2 * C + row));
      uint32_t r[4][4];
      const bool in = row < rows;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (in) lds_v4(s_v + place(row, 4 * half + q), r[q]);
        else r[q][0] = r[q][1] = r[q][2] = r[q][3] = 0u;
      }
      float f = w;
      if constexpr (F16) {
        __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(*reinterpret_cast<__half2*>(&r[q][e])));
        const float big = group_max(fminf(fmaxf(__low2float(top), __high2float(top)), 65504.f) * w, c & 1);
        if (!ok) return;
        const int e = max(min(exponent(big) - 14, 100), -100);
        f = w * pow2(-e);
        back_next = pow2(e);
      }
      if (!in) {  // behind the sequence
        const uint32_t z[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int q = 0; q < 4; ++q) sts_v4(s_v + place(row, 4 * half + q), z);
#pragma unroll
        for (int q = 0; q < 8; ++q) sts_v4(s_k + half * TILE + place(row, q), z);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w4[S::NV][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t pieces[S::NV];
          split<T, S::NV>(Act<T>::get(r[q][e], 0) * f, Act<T>::get(r[q][e], 1) * f, pieces);
#pragma unroll
          for (int k = 0; k < S::NV; ++k) w4[k][e] = pieces[k];
        }
#pragma unroll
        for (int k = 0; k < S::NV; ++k) sts_v4(to + k * TILE + place(row, 4 * half + q), w4[k]);
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S::VF, c & 1));
    };
    if (chunks > 0) {
      if constexpr (!STATES) publish(0);
      if (ok) decayed(0);
    }
    for (int c = 0; c < chunks && ok; ++c) {
      const int i = c & 1;
      back = back_next;
      const float a = lds_f32(decays(c) + 12 * C);
      if (c + 1 < chunks) {
        decayed(c + 1);
        if (!ok) break;
      }
      ok = warp_wait(bar(S::DS, i), (uint32_t)((c >> 1) & 1));
      if constexpr (F16) ok = group_and(ok);  // no warp leaves while another waits at the group's barrier
      if (!ok) break;
      after_sync();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tbase + lanes + T_DS + 64 * i + 32 * k, r);
        tmem_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) st[32 * k + j] = fmaf(a, st[32 * k + j], F16 ? __uint_as_float(r[j]) * back : __uint_as_float(r[j]));
      }
      if constexpr (STATES) {
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::SF, i));
      } else if (c + 1 < chunks) {
        if (c >= 1) ok &= warp_wait(bar(S::OF, i ^ 1), (uint32_t)(((c - 1) >> 1) & 1));
        if (!F16 && !ok) break;
        publish(c + 1);
      }
    }
    if (ok) {
      if constexpr (STATES) {
        float4* to = reinterpret_cast<float4*>(seg.states + (size_t)blockIdx.y * gridDim.x * 128 * VT + tile);
#pragma unroll
        for (int j = 0; j < VT; j += 4) to[(j / 4) * 128 + d] = make_float4(st[j], st[j + 1], st[j + 2], st[j + 3]);
      } else if (p.final_state != nullptr && (int)blockIdx.y == (n > 0 ? (n - 1) / seg.tokens : 0) && d < p.K) {
        float* to = p.final_state + ((size_t)bh * p.K + d) * p.V + v0;
#pragma unroll
        for (int j = 0; j < VT; ++j)
          if (j < cols) to[j] = st[j];
      }
    }
  }
  if (!ok && lane == 0 && p.status != nullptr) atomicExch(p.status, 1);
  __syncwarp();
  before_sync();
  __syncthreads();
  if (warp == ISSUER) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "r"(512u) : "memory");
}

// rows of `width` channels as boxes of 64 tokens x 64 channels, zero behind the last channel and token
static int encode(CUtensorMap* m, bool f16, const void* base, int width, int T, int heads, int B, long long st, long long sh, long long sb) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return fail(LQ_ERR_LAUNCH, "linear_attention: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t gdim[4] = {(cuuint64_t)width, (cuuint64_t)T, (cuuint64_t)heads, (cuuint64_t)B};
  // an axis of one has any stride
  const cuuint64_t gstride[3] = {T > 1 ? (cuuint64_t)st * 2 : 1024, heads > 1 ? (cuuint64_t)sh * 2 : 1024, B > 1 ? (cuuint64_t)sb * 2 : 1024};
  const cuuint32_t box[4] = {64, (cuuint32_t)C, 1, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), gdim, gstride, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LQ_OK : fail(LQ_ERR_LAUNCH, "linear_attention: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

template <typename T>
static int run(const lq_attention_problem* p, const Plan& r, const Segments& seg, cudaStream_t st) {
  using S = Shape<T>;
  CUtensorMap q, k, v;
  if (int e = encode(&q, S::F16, p->q, p->K, p->T, p->Hk, p->B, p->q_stride_t, p->q_stride_h, p->q_stride_b)) return e;
  if (int e = encode(&k, S::F16, p->k, p->K, p->T, p->Hk, p->B, p->k_stride_t, p->k_stride_h, p->k_stride_b)) return e;
  if (int e = encode(&v, S::F16, p->v, p->V, p->T, p->H, p->B, p->v_stride_t, p->v_stride_h, p->v_stride_b)) return e;
  const int wide = p->V % 8 == 0 && (reinterpret_cast<uintptr_t>(p->o) & 15u) == 0;
  const dim3 block(32 * WARPS);
  cudaError_t e = cudaSuccess;
  if (seg.count > 1) {
    e = launch_opt_in(linear_attention_tc_kernel<T, true>, dim3((unsigned)r.tiles, seg.count - 1), block, S::SMEM, st, q, k, v, *p, seg, wide);
    if (e == cudaSuccess && seg.count > 2) e = launch_segment_states(seg, p->B * p->H, r.tiles * 128 * VT, st);
  }
  if (e == cudaSuccess) e = launch_opt_in(linear_attention_tc_kernel<T, false>, dim3((unsigned)r.tiles, seg.count), block, S::SMEM, st, q, k, v, *p, seg, wide);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "linear_attention: %s", cudaGetErrorString(e));
  return check_launch("linear_attention_tc_kernel");
}

}  // namespace attentiontc

namespace attention {

// 16-bit operands whose rows TMA can fetch: every start on a 16-byte boundary, strides that move forwards
bool tc_applies(const lq_attention_problem* p) {
  if (p->dtype == LQ_F32 || p->K > 128 || p->T < 1) return false;
  auto rows = [&](const void* base, int heads, long long st, long long sh, long long sb) {
    auto fits = [](int extent, long long stride) { return extent <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
    return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && fits(p->T, st) && fits(heads, sh) && fits(p->B, sb);
  };
  return rows(p->q, p->Hk, p->q_stride_t, p->q_stride_h, p->q_stride_b) && rows(p->k, p->Hk, p->k_stride_t, p->k_stride_h, p->k_stride_b) &&
         rows(p->v, p->H, p->v_stride_t, p->v_stride_h, p->v_stride_b);
}

int run_tc(const lq_attention_problem* p, const Plan& r, const Segments& seg, cudaStream_t st) {
  return p->dtype == LQ_F16 ? attentiontc::run<__half>(p, r, seg, st) : attentiontc::run<__nv_bfloat16>(p, r, seg, st);
}

}  // namespace attention

}  // namespace lq
