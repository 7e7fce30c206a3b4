// INT8 matrix product on the Blackwell tensor cores: y[m,n] = (sum_k x[m,k] w[n,k]) x_scale[m] w_scale[n] + bias[n].
//
// Persistent kernel, one CTA per SM, tiles of 128 tokens x BN output channels. Both operands are codes with the reduction
// index contiguous: TMA brings blocks of 128 bytes of K (128-byte swizzle, zero-filled behind the last row and the last byte
// of K) into a ring of stages, one thread issues tcgen05.mma.kind::i8 (M = 128, N = BN, four steps of 32 per stage) into one
// of two accumulators in tensor memory, and eight warps turn the other one into outputs meanwhile: INT32 to fp32, both scales
// and the bias, through a swizzled 64-byte row per lane in shared memory, stored as pieces of 64 bytes a row.
// Every wait is bounded; on expiry the CTA raises the status word, lets its copies and products land, frees its tensor
// memory and returns.
#include "lq_layer.cuh"
#include "lq_tc.cuh"

namespace lq {

namespace lineartc {

constexpr int BM = 128, BK = 128, OUT_WARPS = 8, THREADS = 32 * (OUT_WARPS + 2), STAGE_BYTES = 192 * 1024;

template <int BN>
struct Shape {
  static constexpr int STAGE = (BM + BN) * BK, STAGES = STAGE_BYTES / STAGE;
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

template <int BN, typename TO>
__global__ void __launch_bounds__(THREADS, 1) int8_linear_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                    const lq_linear_problem p) {
  using S = Shape<BN>;
  extern __shared__ uint8_t smem_dyn[];
  const uint32_t s_stage = (smem_u32(smem_dyn) + 1023u) & ~1023u, s_out = s_stage + S::STAGES * S::STAGE, s_cols = s_out + S::OUT;
  const uint32_t s_full = s_cols + S::COLS, s_empty = s_full + 8 * S::STAGES, s_acc = s_empty + 8 * S::STAGES, s_free = s_acc + 16, s_tbase = s_free + 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mt = (p.M + BM - 1) / BM, nt = (p.N + BN - 1) / BN, tiles = mt * nt, kblocks = (p.K + BK - 1) / BK;

  pdl_enter();
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_acc + 8 * i, 1);
      mbar_init(s_free + 8 * i, OUT_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == OUT_WARPS + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(s_tbase), "r"((uint32_t)(2 * BN)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tbase = lds_u32(s_tbase);
  bool ok = true;

  if (warp == OUT_WARPS) {  // loads
    if (lane == 0) {
      long long fill = 0;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int m, n;
        tile_at(t, mt, nt, m, n);
        for (int kb = 0; kb < kblocks; ++kb, ++fill) {
          const int s = (int)(fill % S::STAGES);
          if (fill >= S::STAGES && !(ok = mbar_wait_bounded(s_empty + 8 * s, (uint32_t)((fill / S::STAGES + 1) & 1)))) break;
          mbar_expect(s_full + 8 * s, S::STAGE);
          tma_load_2d(s_stage + s * S::STAGE, &map_x, kb * BK, m * BM, s_full + 8 * s);
          tma_load_2d(s_stage + s * S::STAGE + BM * BK, &map_w, kb * BK, n * BN, s_full + 8 * s);
        }
      }
      for (long long f = fill > S::STAGES ? fill - S::STAGES : 0; f < fill; ++f)  // nothing may land after the CTA has gone
        ok &= mbar_wait_bounded(s_full + 8 * (int)(f % S::STAGES), (uint32_t)((f / S::STAGES) & 1));
    }
  } else if (warp == OUT_WARPS + 1) {  // products
    if (lane == 0) {
      const uint32_t idesc = idesc_i8(BM, BN);
      long long fill = 0;
      int i = 0;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
        const int acc = i & 1;
        if (i >= 2 && !(ok = mbar_wait_bounded(s_free + 8 * acc, (uint32_t)((i / 2 + 1) & 1)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        for (int kb = 0; kb < kblocks; ++kb, ++fill) {
          const int s = (int)(fill % S::STAGES);
          if (!(ok = mbar_wait_bounded(s_full + 8 * s, (uint32_t)((fill / S::STAGES) & 1)))) break;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const uint64_t da = desc_kmajor_sw128(s_stage + s * S::STAGE), db = desc_kmajor_sw128(s_stage + s * S::STAGE + BM * BK);
#pragma unroll
          for (int ks = 0; ks < BK / 32; ++ks) umma_i8(tbase + acc * BN, da + 2 * ks, db + 2 * ks, idesc, (kb | ks) > 0);
          umma_commit(s_empty + 8 * s);
        }
        if (!ok) break;
        umma_commit(s_acc + 8 * acc);
      }
      if (!ok && fill > 0)  // the products that were issued: each stage's commit
        for (long long f = fill > S::STAGES ? fill - S::STAGES : 0; f < fill; ++f)
          mbar_wait_bounded(s_empty + 8 * (int)(f % S::STAGES), (uint32_t)((f / S::STAGES) & 1));
    }
  } else {  // outputs: warp w has the accumulator rows 32 (w & 3) .. and half of the columns
    constexpr int CHUNK = 64 / sizeof(TO), PER = 16 / sizeof(TO);  // columns of a 64-byte piece of a row, of 16 bytes
    const int quad = warp & 3, half = (warp >> 2) * S::HALF;
    const uint32_t out = s_out + warp * 32 * 64, cols = s_cols + warp * 2 * S::HALF * 4;
    const bool wide = ((size_t)p.N * sizeof(TO)) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      int m, n;
      tile_at(t, mt, nt, m, n);
      const int acc = i & 1, row0 = m * BM + 32 * quad, n0 = n * BN + half;
      const float xs = row0 + lane < p.M ? __ldg(p.x_scale + row0 + lane) : 0.f;
      __syncwarp();
#pragma unroll
      for (int c = lane; c < S::HALF; c += 32) {
        const bool in = n0 + c < p.N;
        sts_u32(cols + 4 * c, __float_as_uint(in ? __ldg(p.w_scale + n0 + c) : 0.f));
        sts_u32(cols + 4 * (S::HALF + c), __float_as_uint(in && p.bias ? __ldg(p.bias + n0 + c) : 0.f));
      }
      __syncwarp();
      if (!(ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_acc + 8 * acc, (uint32_t)((i / 2) & 1))))) break;
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
      if (lane == 0) mbar_arrive(s_free + 8 * acc);
    }
  }
  if (!ok && p.status != nullptr) atomicExch(p.status, 1);
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if (warp == OUT_WARPS + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "r"((uint32_t)(2 * BN)) : "memory");
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

template <int BN, typename TO>
static int launch_tc(const lq_linear_problem* p, cudaStream_t st) {
  CUtensorMap mx, mw;
  if (int e = encode(&mx, p->x, p->K, p->x_stride, p->M, BM)) return e;
  if (int e = encode(&mw, p->w, p->K, p->w_stride, p->N, BN)) return e;
  const long long tiles = (long long)((p->M + BM - 1) / BM) * ((p->N + BN - 1) / BN);
  if (tiles >= 1ll << 30) return fail(LQ_ERR_SHAPE, "int8_linear: M=%d N=%d", p->M, p->N);
  const int sms = sm_count();
  const cudaError_t e = launch_opt_in(int8_linear_tc_kernel<BN, TO>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(THREADS), Shape<BN>::SMEM, st, mx, mw, *p);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "int8_linear: %s", cudaGetErrorString(e));
  return check_launch("int8_linear_tc_kernel");
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
  return with_dtype(p->out_dtype, "int8_linear", [&](auto t) {
    using TO = decltype(t);
    return best == 256 ? lineartc::launch_tc<256, TO>(p, st) : best == 128 ? lineartc::launch_tc<128, TO>(p, st) : lineartc::launch_tc<64, TO>(p, st);
  });
}

}  // namespace lq
