// INT8 matrix product on the Blackwell tensor cores: y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n].
//
// Persistent kernel, one CTA per SM, tiles of 128 tokens x BN output channels; for many tiles two CTAs of a cluster share one of
// 256 x 256 (tcgen05 cta_group::2: each brings its tokens and half of the weights, the first issues the products of both). Both
// operands are codes with the reduction index contiguous: TMA brings blocks of 128 bytes of K (128-byte swizzle, zero-filled
// behind the last row and the last byte of K) into a ring of stages, one thread issues tcgen05.mma.kind::i8 (four steps of 32 per
// stage) into one of two accumulators in tensor memory, and eight warps turn the other one into outputs meanwhile: INT32 to fp32,
// both scales and the bias, through a swizzled 64-byte row per lane in shared memory, stored as pieces of 64 bytes a row.
// Bound by the tensor pipe: 8192^3 339 us (3.24 POP/s; 366 us without pairs), 32768 x 2560 -> 10576 654 to 705 us (2.7 to 2.5, by the box's power), where what
// torch's INT8 product reaches is 2.94 with INT32 outputs and no scales.
// Every wait is bounded; on expiry the CTA raises the status word, lets its copies and products land, frees its tensor
// memory and returns.
#include "lq_layer.cuh"
#include "lq_tc.cuh"

namespace lq {

namespace lineartc {

constexpr int BM = 128, BK = 128, OUT_WARPS = 8, THREADS = 32 * (OUT_WARPS + 2), STAGE_BYTES = 192 * 1024;

// PAIR: two CTAs of a cluster on one tile of 256 tokens, each with 128 of them and half of the weights' rows
template <int BN, bool PAIR>
struct Shape {
  static constexpr int WROWS = PAIR ? BN / 2 : BN, STAGE = (BM + WROWS) * BK, STAGES = STAGE_BYTES / STAGE;
  static constexpr int HALF = BN / 2;                                     // columns of a storing warp: two share 32 rows
  static constexpr int OUT = OUT_WARPS * 32 * 64, COLS = OUT_WARPS * 2 * HALF * 4;  // per storing warp: 32 rows of 64 bytes; w_scale and bias of its columns
  static constexpr int BARS = (2 * STAGES + 4) * 8;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + OUT + COLS + BARS + 16;
};

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts_u4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ---- one CTA, or a pair of a cluster
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t in_first(uint32_t addr) {  // the same place in the pair's first CTA
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(a) : "r"(addr));
  return a;
}
__device__ __forceinline__ void mbar_arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(in_first(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity) {  // what the other CTA did before it arrived is visible
  for (int it = 0; it < (1 << 20); ++it) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(in_first(bar))
                 : "memory");
  else tma_load_2d(dst, map, c0, c1, bar);
}
template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
  else umma_i8(d, a, b, idesc, accumulate);
}
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {  // of a pair: the barriers of both
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else umma_commit(bar);
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t from, uint32_t columns) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(from), "r"(columns) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(from), "r"(columns) : "memory");
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Tiles of up to 16 row blocks share the weights of a column block before the next column block is taken
__device__ __forceinline__ void tile_at(int t, int mt, int nt, int& m, int& n) {
  constexpr int GROUP = 16;
  const int g = t / (GROUP * nt), in = t - g * GROUP * nt, rows = min(GROUP, mt - g * GROUP);
  n = in / rows;
  m = g * GROUP + in - n * rows;
}

template <int BN, bool PAIR, typename TO>
__global__ void __launch_bounds__(THREADS, 1) int8_linear_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                    const lq_linear_problem p) {
  using S = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_dyn[];
  const uint32_t s_stage = (smem_u32(smem_dyn) + 1023u) & ~1023u, s_out = s_stage + S::STAGES * S::STAGE, s_cols = s_out + S::OUT;
  const uint32_t s_full = s_cols + S::COLS, s_empty = s_full + 8 * S::STAGES, s_acc = s_empty + 8 * S::STAGES, s_free = s_acc + 16, s_tbase = s_free + 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0, first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  const int mt = (p.M + CTAS * BM - 1) / (CTAS * BM), nt = (p.N + BN - 1) / BN, tiles = mt * nt, kblocks = (p.K + BK - 1) / BK;

  pdl_enter();
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_acc + 8 * i, 1);
      mbar_init(s_free + 8 * i, CTAS * OUT_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == OUT_WARPS + 1) tmem_alloc<PAIR>(s_tbase, 2 * BN);
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are there
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tbase = lds_u32(s_tbase);
  bool ok = true;

  // a stage and how often it has been filled before, without a division per block
  struct Ring {
    int s = 0;
    uint32_t lap = 0;
    __device__ __forceinline__ void next() {
      if (++s == S::STAGES) s = 0, ++lap;
    }
  };
  auto wait = [&](uint32_t bar, uint32_t parity) { return PAIR ? mbar_wait_cluster(bar, parity) : mbar_wait_bounded(bar, parity); };
  if (warp == OUT_WARPS) {  // loads; of a pair, all arrive at the first CTA's barriers
    if (lane == 0) {
      Ring r;
      for (int t = first; t < tiles && ok; t += step) {
        int m, n;
        tile_at(t, mt, nt, m, n);
        const int row = (m * CTAS + rank) * BM, col = n * BN + rank * S::WROWS;
        for (int kb = 0; kb < kblocks; ++kb, r.next()) {
          if (r.lap > 0 && !(ok = wait(s_empty + 8 * r.s, (r.lap + 1) & 1))) break;
          if (rank == 0) mbar_expect(s_full + 8 * r.s, CTAS * S::STAGE);
          tma_load<PAIR>(s_stage + r.s * S::STAGE, &map_x, kb * BK, row, s_full + 8 * r.s);
          tma_load<PAIR>(s_stage + r.s * S::STAGE + BM * BK, &map_w, kb * BK, col, s_full + 8 * r.s);
        }
      }
      if (rank == 0)
        for (int i = 0; i < S::STAGES; ++i, r.next())  // nothing may land after the CTA has gone: the last fill of each stage
          if (r.lap > 0) ok &= wait(s_full + 8 * r.s, (r.lap + 1) & 1);
    }
  } else if (warp == OUT_WARPS + 1) {  // products
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_i8(CTAS * BM, BN);
      Ring r;
      int i = 0;
      for (int t = first; t < tiles && ok; t += step, ++i) {
        const int acc = i & 1;
        if (i >= 2 && !(ok = wait(s_free + 8 * acc, (uint32_t)((i / 2 + 1) & 1)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        for (int kb = 0; kb < kblocks; ++kb, r.next()) {
          if (!(ok = wait(s_full + 8 * r.s, r.lap & 1))) break;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const uint64_t da = desc_kmajor_sw128(s_stage + r.s * S::STAGE), db = desc_kmajor_sw128(s_stage + r.s * S::STAGE + BM * BK);
#pragma unroll
          for (int ks = 0; ks < BK / 32; ++ks) mma<PAIR>(tbase + acc * BN, da + 2 * ks, db + 2 * ks, idesc, (kb | ks) > 0);
          commit<PAIR>(s_empty + 8 * r.s);
        }
        if (!ok) break;
        commit<PAIR>(s_acc + 8 * acc);
      }
      if (!ok)  // the products that were issued: each stage's commit
        for (int k = 0; k < S::STAGES; ++k, r.next())
          if (r.lap > 0) wait(s_empty + 8 * r.s, (r.lap + 1) & 1);
    }
  } else {  // outputs: warp w has the accumulator rows 32 (w & 3) .. and half of the columns
    constexpr int CHUNK = 64 / sizeof(TO), PER = 16 / sizeof(TO);  // columns of a 64-byte piece of a row, of 16 bytes
    const int quad = warp & 3, half = (warp >> 2) * S::HALF;
    const uint32_t out = s_out + warp * 32 * 64, cols = s_cols + warp * 2 * S::HALF * 4;
    const bool wide = ((size_t)p.N * sizeof(TO)) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
    int i = 0;
    for (int t = first; t < tiles; t += step, ++i) {
      int m, n;
      tile_at(t, mt, nt, m, n);
      const int acc = i & 1, row0 = (m * CTAS + rank) * BM + 32 * quad, n0 = n * BN + half;
      const float xs = row0 + lane < p.M ? __ldg(p.x_scale + row0 + lane) : 0.f;
      __syncwarp();
#pragma unroll
      for (int c = lane; c < S::HALF; c += 32) {
        const bool in = n0 + c < p.N;
        sts_u32(cols + 4 * c, __float_as_uint(in ? __ldg(p.w_scale + n0 + c) : 0.f));
        sts_u32(cols + 4 * (S::HALF + c), __float_as_uint(in && p.bias ? __ldg(p.bias + n0 + c) : 0.f));
      }
      __syncwarp();
      if (!(ok = __all_sync(0xffffffffu, wait(s_acc + 8 * acc, (uint32_t)((i / 2) & 1))))) break;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll 1
      for (int c0 = 0; c0 < S::HALF; c0 += CHUNK) {
        if (n0 + c0 >= p.N) break;
        uint32_t r[CHUNK];
        const uint32_t from = tbase + ((uint32_t)(32 * quad) << 16) + acc * BN + half + c0;
        if constexpr (CHUNK == 32) tmem_ld_32x32b_x32(from, r);
        else tmem_ld_32x32b_x16(from, r);
        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        float v[CHUNK];
#pragma unroll
        for (int j = 0; j < CHUNK; j += 4) {
          const float4 ws = lds_f4(cols + 4 * (c0 + j)), b = lds_f4(cols + 4 * (S::HALF + c0 + j));
          v[j] = fmaf((float)(int)r[j] * xs, ws.x, b.x);
          v[j + 1] = fmaf((float)(int)r[j + 1] * xs, ws.y, b.y);
          v[j + 2] = fmaf((float)(int)r[j + 2] * xs, ws.z, b.z);
          v[j + 3] = fmaf((float)(int)r[j + 3] * xs, ws.w, b.w);
        }
        __syncwarp();  // the chunk before has been read
        // rows of 64 bytes, pairs of them on the same banks: a piece at its place exclusive-or half the row's number
        auto place = [](int row, int piece) { return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4); };
#pragma unroll
        for (int j = 0; j < CHUNK; j += PER) {
          uint4 w;
          if constexpr (sizeof(TO) == 4) {
            w = make_uint4(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3]));
          } else {
            w = make_uint4(Act<TO>::pack2(v[j], v[j + 1]), Act<TO>::pack2(v[j + 2], v[j + 3]), Act<TO>::pack2(v[j + 4], v[j + 5]),
                           Act<TO>::pack2(v[j + 6], v[j + 7]));
          }
          sts_u4(out + place(lane, j / PER), w);
        }
        __syncwarp();
        TO* y = reinterpret_cast<TO*>(p.y);
        if (wide) {
          const int piece = lane & 3, c = n0 + c0 + piece * PER;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int row = 8 * q + (lane >> 2);
            const uint4 w = lds_u4(out + place(row, piece));
            if (row0 + row < p.M && c < p.N) *reinterpret_cast<uint4*>(y + (size_t)(row0 + row) * p.N + c) = w;
          }
        } else {  // rows off 16-byte boundaries: consecutive values a store
          constexpr int ROWS = 32 / CHUNK;
          const int e = lane % CHUNK, byte = e * (int)sizeof(TO);
          for (int q = 0; q < 32; q += ROWS) {
            const int row = q + lane / CHUNK;
            const uint32_t a = out + place(row, byte >> 4) + (byte & 15);
            if (row0 + row < p.M && n0 + c0 + e < p.N) {
              if constexpr (sizeof(TO) == 4) {
                y[(size_t)(row0 + row) * p.N + n0 + c0 + e] = __uint_as_float(lds_u32(a));
              } else {
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(w) : "r"(a));
                reinterpret_cast<uint16_t*>(y)[(size_t)(row0 + row) * p.N + n0 + c0 + e] = w;
              }
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_first(s_free + 8 * acc);
        else mbar_arrive(s_free + 8 * acc);
      }
    }
  }
  if (!ok && p.status != nullptr) atomicExch(p.status, 1);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // neither CTA's memory is used by the other any more
  if (warp == OUT_WARPS + 1) tmem_free<PAIR>(tbase, 2 * BN);
}

// ---- few tiles: the CTAs of a cluster take parts of K
// Their INT32 sums meet in shared memory, each CTA adds and scales a share of the tile's rows: the sum of integers is the same
// in any order, and no workspace is needed. A ring of 96 KB leaves room for two CTAs on an SM.
struct Split {
  static constexpr int BN = 64, STAGE = (BM + BN) * BK, STAGES = 4, PITCH = BN * 4 + 16;  // rows of the sums on odd multiples of 16 bytes
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + (2 * STAGES + 1) * 8 + 8;
  static_assert(BM * PITCH <= STAGES * STAGE);
};

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ int4 ld_cluster(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <typename TO>
__global__ void __launch_bounds__(THREADS, 2) int8_linear_split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                       const lq_linear_problem p, int parts) {
  using S = Split;
  extern __shared__ uint8_t smem_dyn[];
  const uint32_t s_stage = (smem_u32(smem_dyn) + 1023u) & ~1023u, s_full = s_stage + S::STAGES * S::STAGE, s_empty = s_full + 8 * S::STAGES;
  const uint32_t s_acc = s_empty + 8 * S::STAGES, s_tbase = s_acc + 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_rank(), tile = blockIdx.x / parts;
  const int nt = (p.N + S::BN - 1) / S::BN, m0 = tile / nt * BM, n0 = tile % nt * S::BN, rows = min(BM, p.M - m0);
  const int kblocks = (p.K + BK - 1) / BK, kb0 = kblocks * rank / parts, count = kblocks * (rank + 1) / parts - kb0;

  pdl_enter();
  if (tid == 0) {
    for (int i = 0; i < 2 * S::STAGES + 1; ++i) mbar_init(s_full + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == OUT_WARPS + 1) tmem_alloc<false>(s_tbase, S::BN);
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tbase = lds_u32(s_tbase);
  bool ok = true;
  // thread tid adds the pieces rank 256 + tid + 256 parts i of four columns: the same columns each time
  constexpr int PIECES = S::BN / 4, MOST = BM * PIECES / (2 * 32 * OUT_WARPS);
  const int c = tid % PIECES * 4, row0 = rank * (32 * OUT_WARPS / PIECES) + tid / PIECES, rows_a_round = parts * (32 * OUT_WARPS / PIECES);
  float ws[4], bias[4], xs[MOST];

  if (warp == OUT_WARPS) {
    if (lane == 0) {
      int k = 0;
      for (; k < count; ++k) {
        const int s = k % S::STAGES, lap = k / S::STAGES;
        if (lap > 0 && !(ok = mbar_wait_bounded(s_empty + 8 * s, (lap + 1) & 1))) break;
        mbar_expect(s_full + 8 * s, S::STAGE);
        tma_load_2d(s_stage + s * S::STAGE, &map_x, (kb0 + k) * BK, m0, s_full + 8 * s);
        tma_load_2d(s_stage + s * S::STAGE + BM * BK, &map_w, (kb0 + k) * BK, n0, s_full + 8 * s);
      }
      for (int s = 0; s < min(k, S::STAGES); ++s)  // nothing may land after the CTA has gone: the last fill of each stage
        ok &= mbar_wait_bounded(s_full + 8 * s, (k - 1 - s) / S::STAGES & 1);
    }
  } else if (warp == OUT_WARPS + 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_i8(BM, S::BN);
      for (int k = 0; k < count; ++k) {
        const int s = k % S::STAGES, lap = k / S::STAGES;
        if (!(ok = mbar_wait_bounded(s_full + 8 * s, lap & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const uint64_t da = desc_kmajor_sw128(s_stage + s * S::STAGE), db = desc_kmajor_sw128(s_stage + s * S::STAGE + BM * BK);
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) umma_i8(tbase, da + 2 * ks, db + 2 * ks, idesc, (k | ks) > 0);
        umma_commit(s_empty + 8 * s);
      }
      umma_commit(s_acc);
    }
  } else {  // sums to shared memory: the stages are free once the last product is done
    const int quad = warp & 3, c0 = (warp >> 2) * 32;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = n0 + c + j < p.N;
      ws[j] = in ? __ldg(p.w_scale + n0 + c + j) : 0.f;
      bias[j] = in && p.bias ? __ldg(p.bias + n0 + c + j) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < MOST; ++i) xs[i] = row0 + i * rows_a_round < rows ? __ldg(p.x_scale + m0 + row0 + i * rows_a_round) : 0.f;
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_acc, 0));
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (ok && 32 * quad < rows) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(tbase + ((uint32_t)(32 * quad) << 16) + c0, r);
      asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
      for (int j = 0; j < 32; j += 4) sts_u4(s_stage + (32 * quad + lane) * S::PITCH + 4 * (c0 + j), make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]));
    }
  }
  if (!ok && p.status != nullptr) atomicExch(p.status, 1);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync();  // the sums of all are there
  if (warp == OUT_WARPS + 1) tmem_free<false>(tbase, S::BN);
  else if (warp < OUT_WARPS) {
    TO* y = reinterpret_cast<TO*>(p.y);
    const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(TO) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int row = row0 + i * rows_a_round, n = n0 + c;
      if (row >= rows || n >= p.N) continue;
      int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll 4
      for (int q = 0; q < parts; ++q) {
        const int4 v = ld_cluster(in_cta(s_stage + row * S::PITCH + 4 * c, q));
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      const float f[4] = {fmaf((float)sum.x * xs[i], ws[0], bias[0]), fmaf((float)sum.y * xs[i], ws[1], bias[1]), fmaf((float)sum.z * xs[i], ws[2], bias[2]),
                          fmaf((float)sum.w * xs[i], ws[3], bias[3])};
      TO* to = y + (size_t)(m0 + row) * p.N + n;
      if (wide) {
        Pack<TO, 4> out;
        out.set(f);
        store_pack(to, out);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) to[j] = from_f32<TO>(f[j]);
      }
    }
  }
  __syncwarp();
  cluster_sync();  // no CTA reads another's sums any more
}

static int encode(CUtensorMap* m, const void* base, long long row_bytes, long long pitch, long long rows, int box_rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return fail(LQ_ERR_LAUNCH, "int8_linear: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t gdim[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
  const cuuint64_t gstride[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LQ_OK : fail(LQ_ERR_LAUNCH, "int8_linear: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

template <typename... KArgs, typename... Args>
static int launch_clusters(void (*kern)(KArgs...), int ctas, int cluster, size_t smem, cudaStream_t st, Args&&... args) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, args...);
  }
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "int8_linear: %s", cudaGetErrorString(e));
  return check_launch("int8_linear");
}

template <int BN, bool PAIR, typename TO>
static int launch_tc(const lq_linear_problem* p, cudaStream_t st) {
  using S = Shape<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  CUtensorMap mx, mw;
  if (int e = encode(&mx, p->x, p->K, p->x_stride, p->M, BM)) return e;
  if (int e = encode(&mw, p->w, p->K, p->w_stride, p->N, S::WROWS)) return e;
  const long long tiles = (long long)((p->M + CTAS * BM - 1) / (CTAS * BM)) * ((p->N + BN - 1) / BN);
  if (tiles >= 1ll << 29) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d N=%d", p->M, p->N);
  const int units = sm_count() / CTAS;
  return launch_clusters(int8_linear_tc_kernel<BN, PAIR, TO>, CTAS * (int)(tiles < units ? tiles : units), CTAS, S::SMEM, st, mx, mw, *p);
}

template <typename TO>
static int launch_split(const lq_linear_problem* p, int tiles, int parts, cudaStream_t st) {
  CUtensorMap mx, mw;
  if (int e = encode(&mx, p->x, p->K, p->x_stride, p->M, BM)) return e;
  if (int e = encode(&mw, p->w, p->K, p->w_stride, p->N, Split::BN)) return e;
  return launch_clusters(int8_linear_split_kernel<TO>, tiles * parts, parts, Split::SMEM, st, mx, mw, *p, parts);
}

}  // namespace lineartc

// The widest tiles that do not leave SMs idle: rounds of tiles x the time of one, which grows with its width and a fixed part
// (the 128 rows of x that every tile loads)
int run_linear_tc(const lq_linear_problem* p, cudaStream_t st) {
  const long long mt = (p->M + 127) / 128, sms = sm_count();
  int best = 256;
  long long least = 0;
  for (int bn = 256; bn >= 64; bn /= 2) {
    const long long rounds = (mt * ((p->N + bn - 1) / bn) + sms - 1) / sms, cost = rounds * (bn + 64);
    if (least == 0 || cost < least) best = bn, least = cost;
  }
  // Pairs of CTAs read the weights half as often from shared memory; over a few rounds their larger tiles cost more than that:
  // 8192 x 2560 -> 2560 (4.3 rounds) 54 us against 53, 4096 x 2560 -> 10576 (9) 91 against 102, 32768 x 2560 -> 10576 (73) 688 against 743
  const bool pair = mt * ((p->N + 255) / 256) >= 6 * sms;
  // Few tiles of a long K: parts of at least 8 blocks for the CTAs of a cluster, two CTAs on an SM. 5120 -> 2560, 64 tokens: one part
  // 14.3 us, 2, 4, 8 parts 11.0, 8.6, 8.7; 256 tokens, 2 parts: 14.5 -> 12.5; 8192 -> 1024, 33 tokens, 8 parts: 20.7 -> 7.9. To meet
  // costs some 2 us, more than a short K has: 200 x 2560 -> 2560 9.0 -> 9.5, 100 x 1024 -> 1024 4.9 -> 6.7
  const long long narrow = mt * ((p->N + lineartc::Split::BN - 1) / lineartc::Split::BN), blocks = (p->K + lineartc::BK - 1) / lineartc::BK;
  int parts = blocks < 32 ? 1 : 8;
  while (parts > 1 && (narrow * parts > 2 * sms || blocks < 8 * parts)) parts /= 2;
  return with_dtype(p->out_dtype, "int8_linear", [&](auto t) {
    using TO = decltype(t);
    if (parts > 1) return lineartc::launch_split<TO>(p, (int)narrow, parts, st);
    if (pair) return lineartc::launch_tc<256, true, TO>(p, st);
    return best == 256 ? lineartc::launch_tc<256, false, TO>(p, st) : best == 128 ? lineartc::launch_tc<128, false, TO>(p, st) : lineartc::launch_tc<64, false, TO>(p, st);
  });
}

}  // namespace lq
