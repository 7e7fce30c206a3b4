// Selective scan over the tokens of a prompt, one decay rate per channel and state.
//
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n],   y_t = sum_n C_t[n] h_t[n] + skip u_t,   y_t *= silu(z_t)
//
// Two resources bound it: the exponentials (one per token, channel and state, 16 a clock and SM) and what shared memory
// delivers to registers (128 bytes a clock and SM, broadcasts included). A thread of the recurrence holds SPT states of a
// channel, LP threads share the channel; tokens go one after the other, four at a time: dt and dt u (16 bytes each), B and C
// of its states (in fp32 up to four states: unpacking costs more issue slots than the bytes cost clocks) and its part of y lie
// with the token index contiguous, so that one access covers the four. Per token a warp takes 3 + 2 SPT clocks of shared memory
// and 2 SPT of exponentials.
// A tile of TT tokens passes three jobs, each with warps of its own, so that their latencies overlap: dt and dt u are
// prepared and B and C turned, the recurrence runs, and y is stored (the sum of the threads' parts, skip and gate). Buffers of
// two, one barrier a tile. Inputs come as TMA tiles into a ring of ST tiles, requested ST - 2 tiles ahead of their use. Where
// rows do not lie on 16-byte boundaries the storing warps copy them in pieces of eight or four bytes, the pieces that hold a
// row's ends included.
// At 1 x 16384 x 2048 with 16 states (bf16, gate): 369 us; 115 us of exponentials, 41 us of bytes. All jobs in every warp took
// 1 139 us, two jobs and plain loads 937 us, three jobs with the state index contiguous 462 us. The recurrence alone takes 259
// us, the other two jobs alone 211 us; together shared memory is busy in 75 % of the clocks.
#include "lq_layer.cuh"
#include "lq_tc.cuh"

namespace lq {

namespace scan {

// RT threads of the recurrence
template <typename T, int RT_, int SPT, int LP, int ST_, int TT_>
struct Shape {
  // The exponent's rounding costs a decay up to |dt A| 2^-24, which a state that only decays collects: 1e-6 of it over 100 tokens
  // of dt A = -0.1. With fp32 inputs expf carries what the product with log2(e) loses; it takes a fifth more time.
  static constexpr bool ACCURATE = sizeof(T) == 4;
  using BT = std::conditional_t<SPT <= 4 || sizeof(T) == 4, float, T>;  // B and C of the recurrence
  static constexpr int RT = RT_, ST = ST_, TT = TT_, JOB = 256, THREADS = RT + 2 * JOB;  // JOB: threads of the preparing and of the storing job
  static constexpr int NP = SPT * LP, CH = RT / LP, PT = TT + 4;        // PT: pitch of a row of tokens, no two rows of an access on one bank
  static constexpr int GSTEP = JOB / CH, GROUPS = TT / 4;               // a job's thread has one channel, every GSTEP-th group of four tokens
  static constexpr int E = sizeof(T), CB = CH * E, NB = NP * E;         // bytes of a row of channels, of states
  static constexpr int CROW = (CB + 31) / 16 * 16, NROW = (NB + 31) / 16 * 16;  // pitch of rows that are copied by words
  static constexpr int STAGE = TT * (3 * CROW + 2 * NROW);
  static constexpr int YC = LP * PT + 4;                                // parts of y of a channel: again on banks of their own
  static_assert(JOB % CH == 0 && CH % 8 == 0, "");
  struct alignas(128) Smem {
    uint8_t raw[ST][STAGE];  // rows of u, dt, z, B, C
    float dt[2][CH * PT], du[2][CH * PT], y[2][CH * YC];  // dt (times log2(e) unless ACCURATE), dt u, parts of y
    BT B[2][NP * PT], C[2][NP * PT];
    uint64_t full[ST];
    float behind[16];        // the recurrence requests up to 16 tokens behind a row
  };
};

struct Maps {
  CUtensorMap u, dt, z, B, C;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
               : "memory");
}

// One input of the CTA in global memory
struct Rows {
  const uint8_t* from;  // row 0 of the sequence
  long long pitch;      // bytes
  // element 0 of a row that was copied by pieces lies this many bytes behind the copy's start
  __device__ __forceinline__ int shift(int t) const { return ((uint32_t)reinterpret_cast<uintptr_t>(from) + (uint32_t)t * (uint32_t)pitch) & 3; }
  // rows of at most MOST bytes at ROW bytes in shared memory, TT of them; eight threads a row. UNIT: bytes of a copy
  template <int JOB, int TT, int ROW, int MOST, int UNIT>
  __device__ __forceinline__ void copy_by(uint32_t to, int bytes, int t0, int len, int tid) const {
    const uint8_t* at = from + (t0 + (tid >> 3)) * pitch;
    to += (tid >> 3) * ROW + (tid & 7) * UNIT;
#pragma unroll
    for (int i = 0; i < (TT + JOB / 8 - 1) / (JOB / 8); ++i, at += JOB / 8 * pitch, to += JOB / 8 * ROW) {
      const int row = (tid >> 3) + i * (JOB / 8);
      if (row >= TT || t0 + row >= len) break;
      const int sh = UNIT == 4 ? (int)((uint32_t)reinterpret_cast<uintptr_t>(at) & 3) : 0, units = (bytes + sh + UNIT - 1) / UNIT;
      const uint8_t* piece = at - sh + (tid & 7) * UNIT;
#pragma unroll
      for (int j = 0; j < (MOST + 3 + UNIT - 1) / UNIT; j += 8)
        if ((tid & 7) + j < units)
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(to + j * UNIT), "l"(piece + j * UNIT), "n"(UNIT) : "memory");
    }
  }
  template <int JOB, int TT, int ROW, int MOST>
  __device__ __forceinline__ void copy(uint32_t to, int bytes, int t0, int len, int tid, bool by8) const {
    if (from == nullptr) return;
    if (by8) copy_by<JOB, TT, ROW, MOST, 8>(to, bytes, t0, len, tid);
    else copy_by<JOB, TT, ROW, MOST, 4>(to, bytes, t0, len, tid);
  }
};

// ---- what the preparing and the storing job share
// WIDE: rows on 16-byte boundaries, TMA tiles
template <typename T, typename S, bool WIDE>
struct Job {
  const lq_scan_problem& p;
  const Maps& maps;
  typename S::Smem& sm;
  const int tid, b, grp, ch0, len, tiles, ch, g0;
  const bool on;  // the thread's channel is one of the group's
  Rows u, dt, z, B, C;

  __device__ __forceinline__ Job(const lq_scan_problem& p, const Maps& maps, typename S::Smem& sm, int tid, int b, int grp, int ch0, int len)
      : p(p), maps(maps), sm(sm), tid(tid), b(b), grp(grp), ch0(ch0), len(len), tiles((len + S::TT - 1) / S::TT), ch(tid % S::CH), g0(tid / S::CH),
        on(ch0 + tid % S::CH < p.D / p.G) {
    const int d = grp * (p.D / p.G) + ch0;
    auto base = [](const void* x, long long elements) { return x ? reinterpret_cast<const uint8_t*>(x) + elements * S::E : nullptr; };
    u = {base(p.u, b * p.u_stride_b + d), p.u_stride_t * S::E};
    dt = {base(p.dt, b * p.dt_stride_b + d), p.dt_stride_t * S::E};
    z = {base(p.z, b * p.z_stride_b + d), p.z_stride_t * S::E};
    B = {base(p.Bm, b * p.B_stride_b + grp * p.B_stride_g), p.B_stride_t * S::E};
    C = {base(p.Cm, b * p.C_stride_b + grp * p.C_stride_g), p.C_stride_t * S::E};
  }
  __device__ __forceinline__ int channel() const { return grp * (p.D / p.G) + ch0 + ch; }
  // where array i of a stage (u, dt, z, B, C) begins, and the pitch of its rows
  static __device__ __forceinline__ constexpr int offset(int i) { return i < 3 ? i * S::TT * S::CROW : 3 * S::TT * S::CROW + (i - 3) * S::TT * S::NROW; }
  static __device__ __forceinline__ constexpr int pitch(int i) { return i < 3 ? (WIDE ? S::CB : S::CROW) : (WIDE ? S::NB : S::NROW); }
  __device__ __forceinline__ const uint8_t* stage(int tile) const { return sm.raw[tile % S::ST]; }
  // element c of row r of array i
  template <int I>
  __device__ __forceinline__ T at(const uint8_t* stage, const Rows& src, int tile, int r, int c) const {
    int o = offset(I) + r * pitch(I) + c * S::E;
    if constexpr (!WIDE) o += src.shift(tile * S::TT + r);
    return *reinterpret_cast<const T*>(stage + o);
  }
};

// ---- dt and dt u of a tile; B and C with the token index contiguous
template <typename T, typename S, bool WIDE>
struct Prepare : Job<T, S, WIDE> {
  using J = Job<T, S, WIDE>;
  using J::p, J::sm, J::tid, J::len, J::ch, J::g0, J::on, J::u, J::dt, J::B, J::C;
  float bias;
  bool ok = true;

  template <typename... A>
  __device__ __forceinline__ Prepare(A&&... a) : J(a...), bias(on && p.dt_bias ? p.dt_bias[J::channel()] : 0.f) {}
  // FULL: every token of the tile counts
  template <bool FULL, bool SOFTPLUS>
  __device__ __forceinline__ void steps(const uint8_t* st, int tile) {
    const int t0 = tile * S::TT, buf = tile & 1;
#pragma unroll
    for (int g = g0; g < S::GROUPS; g += S::GSTEP) {
      float v[4], w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = to_f32(J::template at<1>(st, dt, tile, 4 * g + k, ch)) + bias;
        w[k] = to_f32(J::template at<0>(st, u, tile, 4 * g + k, ch));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = clamp_nan(SOFTPLUS ? softplus<S::ACCURATE>(v[k]) : v[k], p.dt_min, p.dt_max);
        w[k] *= v[k];
        // here and not on A: the rounding of a factor that all tokens share would add up over them
        if constexpr (!S::ACCURATE) v[k] *= kLog2e;
        if (!FULL && t0 + 4 * g + k >= len) v[k] = w[k] = 0.f;  // a token behind the last is a step of nothing
      }
      *reinterpret_cast<float4*>(&sm.dt[buf][ch * S::PT + 4 * g]) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(&sm.du[buf][ch * S::PT + 4 * g]) = make_float4(w[0], w[1], w[2], w[3]);
    }
  }
  template <bool FULL>
  __device__ __forceinline__ void turn(const uint8_t* st, int tile) {
    const int t0 = tile * S::TT, buf = tile & 1;
    const T none = from_f32<T>(0.f);
    constexpr int PER = S::JOB / S::NP, WORK = S::TT / 2;  // pairs of tokens, of a state in PER threads
    const int n = tid % S::NP;
#pragma unroll
    for (int i = 0; i < (WORK + PER - 1) / PER; ++i) {
      const int r = 2 * (tid / S::NP + i * PER);
      if (WORK % PER && r >= S::TT) break;
      // what lies behind the last token or state takes no part, not even as 0 x NaN
      const bool in0 = FULL || (n < p.N && t0 + r < len), in1 = FULL || (n < p.N && t0 + r + 1 < len);
      Pack<typename S::BT, 2> vB, vC;
      vB.v[0] = from_f32<typename S::BT>(to_f32(in0 ? J::template at<3>(st, B, tile, r, n) : none));
      vB.v[1] = from_f32<typename S::BT>(to_f32(in1 ? J::template at<3>(st, B, tile, r + 1, n) : none));
      vC.v[0] = from_f32<typename S::BT>(to_f32(in0 ? J::template at<4>(st, C, tile, r, n) : none));
      vC.v[1] = from_f32<typename S::BT>(to_f32(in1 ? J::template at<4>(st, C, tile, r + 1, n) : none));
      store_pack(&sm.B[buf][n * S::PT + r], vB);
      store_pack(&sm.C[buf][n * S::PT + r], vC);
    }
  }
  __device__ __forceinline__ void run(int tile) {
    if (WIDE && ok) ok = mbar_wait_bounded(smem_u32(&sm.full[tile % S::ST]), (uint32_t)((tile / S::ST) & 1));
    const uint8_t* st = J::stage(tile);
    if (WIDE && (tile + 1) * S::TT <= len) {  // TMA fills with zeros behind the last state
      turn<true>(st, tile);
      if (p.softplus) steps<true, true>(st, tile);
      else steps<true, false>(st, tile);
    } else {
      turn<false>(st, tile);
      if (p.softplus) steps<false, true>(st, tile);
      else steps<false, false>(st, tile);
    }
  }
};

// ---- loads, and y of a tile
template <typename T, typename S, bool WIDE>
struct Store : Job<T, S, WIDE> {
  using J = Job<T, S, WIDE>;
  using J::p, J::maps, J::sm, J::tid, J::len, J::ch, J::g0, J::on, J::u, J::dt, J::z, J::B, J::C;
  const bool by8;  // rows on 8-byte boundaries
  T* y;
  float skip;

  template <typename... A>
  __device__ __forceinline__ Store(bool by8, A&&... a) : J(a...), by8(by8), y(reinterpret_cast<T*>(p.y) + (size_t)J::b * p.T * p.D + J::channel()), skip(on && p.skip ? p.skip[J::channel()] : 0.f) {}
  __device__ __forceinline__ void request(int tile) const {
    const int t0 = tile * S::TT;
    const uint32_t to = smem_u32(J::stage(tile));
    if constexpr (WIDE) {
      if (tid == 0 && tile < J::tiles) {
        const uint32_t bar = smem_u32(&sm.full[tile % S::ST]);
        const int d = J::grp * (p.D / p.G) + J::ch0;
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the stage has been read with plain loads
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((uint32_t)(S::TT * ((p.z ? 3 : 2) * S::CB + 2 * S::NB)))
                     : "memory");
        tma_load_3d(to + J::offset(0), &maps.u, d, t0, J::b, bar);
        tma_load_3d(to + J::offset(1), &maps.dt, d, t0, J::b, bar);
        if (p.z) tma_load_3d(to + J::offset(2), &maps.z, d, t0, J::b, bar);
        tma_load_4d(to + J::offset(3), &maps.B, 0, J::grp, t0, J::b, bar);
        tma_load_4d(to + J::offset(4), &maps.C, 0, J::grp, t0, J::b, bar);
      }
    } else {
      const int bytes = min(S::CH, p.D / p.G - J::ch0) * S::E;
      u.template copy<S::JOB, S::TT, S::CROW, S::CB>(to + J::offset(0), bytes, t0, len, tid, by8);
      dt.template copy<S::JOB, S::TT, S::CROW, S::CB>(to + J::offset(1), bytes, t0, len, tid, by8);
      z.template copy<S::JOB, S::TT, S::CROW, S::CB>(to + J::offset(2), bytes, t0, len, tid, by8);
      B.template copy<S::JOB, S::TT, S::NROW, S::NB>(to + J::offset(3), p.N * S::E, t0, len, tid, by8);
      C.template copy<S::JOB, S::TT, S::NROW, S::NB>(to + J::offset(4), p.N * S::E, t0, len, tid, by8);
      cp_async_commit();
    }
  }
  // tiles up to the ST - 3 newest requests are there for everybody from the next barrier on
  __device__ __forceinline__ void arrived() const {
    if constexpr (!WIDE) cp_async_wait<S::ST - 3>();
  }
  template <int LP, bool FULL, bool GATE>
  __device__ __forceinline__ void outputs(int tile) const {
    const int t0 = tile * S::TT;
    const uint8_t* st = J::stage(tile);
#pragma unroll
    for (int g = g0; g < S::GROUPS; g += S::GSTEP) {
      const float* parts = &sm.y[tile & 1][ch * S::YC + 4 * g];
      float4 q = *reinterpret_cast<const float4*>(parts);
      F2 lo(q.x, q.y), hi(q.z, q.w);
#pragma unroll
      for (int l = 1; l < LP; ++l) {
        q = *reinterpret_cast<const float4*>(parts + l * S::PT);
        lo = add2(lo, F2(q.x, q.y));
        hi = add2(hi, F2(q.z, q.w));
      }
      float s[4];
      lo.get(s[0], s[1]);
      hi.get(s[2], s[3]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = fmaf(skip, to_f32(J::template at<0>(st, u, tile, 4 * g + k, ch)), s[k]);
        if (GATE) s[k] *= silu(to_f32(J::template at<2>(st, z, tile, 4 * g + k, ch)));
      }
      T* to = y + (size_t)(t0 + 4 * g) * p.D;
#pragma unroll
      for (int k = 0; k < 4; ++k, to += p.D)
        if (FULL || t0 + 4 * g + k < p.T) *to = from_f32<T>(FULL || t0 + 4 * g + k < len ? s[k] : 0.f);
    }
  }
  template <int LP>
  __device__ __forceinline__ void run(int tile) const {
    if (!on) return;
    if ((tile + 1) * S::TT <= len) {
      if (p.z) outputs<LP, true, true>(tile);
      else outputs<LP, true, false>(tile);
    } else {
      if (p.z) outputs<LP, false, true>(tile);
      else outputs<LP, false, false>(tile);
    }
  }
  __device__ __forceinline__ void zeros(int t0) const {  // tiles that no token reaches
    if (!on) return;
    for (int t = t0 + g0; t < p.T; t += S::GSTEP) y[(size_t)t * p.D] = from_f32<T>(0.f);
  }
};

// ---- the recurrence of a tile, four tokens at a time. Few warps run it, so one's own instructions have to cover latencies: the
// exponentials of four tokens are taken while the recurrence of the four before runs, their operands requested ahead of that.
template <typename T, typename S, int SPT, int LP>
struct Recurrence {
  struct Operands {
    float4 du;
    Pack<typename S::BT, 4> B[SPT], C[SPT];
  };
  typename S::Smem& sm;
  const int ch, ln;  // states ln, ln + LP, ..
  float A[SPT], h[SPT];

  // of the tile: rows of this thread's channel and first state
  const float *pdt, *pdu;
  const typename S::BT *pB, *pC;
  float* py;

  __device__ __forceinline__ float4 load_dt(int t) const { return *reinterpret_cast<const float4*>(pdt + t); }
  __device__ __forceinline__ void load(Operands& o, int t) const {
    o.du = *reinterpret_cast<const float4*>(pdu + t);
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
      o.B[j] = load_pack<typename S::BT, 4>(pB + j * LP * S::PT + t);
      o.C[j] = load_pack<typename S::BT, 4>(pC + j * LP * S::PT + t);
    }
  }
  __device__ __forceinline__ void decays(float (&a)[SPT][4], const float4& dt) const {
    const float t[4] = {dt.x, dt.y, dt.z, dt.w};
#pragma unroll
    for (int j = 0; j < SPT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) a[j][k] = S::ACCURATE ? expf(t[k] * A[j]) : ex2(t[k] * A[j]);
  }
  __device__ __forceinline__ void run(const Operands& o, const float (&a)[SPT][4], int t) {
    const float du[4] = {o.du.x, o.du.y, o.du.z, o.du.w};
    float y[4];
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
      float b[4], c[4];
      o.B[j].get(b);
      o.C[j].get(c);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[j] = fmaf(a[j][k], h[j], du[k] * b[k]);
        y[k] = j == 0 ? h[j] * c[k] : fmaf(h[j], c[k], y[k]);
      }
    }
    *reinterpret_cast<float4*>(py + t) = make_float4(y[0], y[1], y[2], y[3]);
  }
  __device__ __forceinline__ void tile(int buf) {
    pdt = &sm.dt[buf][ch * S::PT];
    pdu = &sm.du[buf][ch * S::PT];
    pB = &sm.B[buf][ln * S::PT];
    pC = &sm.C[buf][ln * S::PT];
    py = &sm.y[buf][ch * S::YC + ln * S::PT];
    if constexpr (SPT <= 2) {
      Operands x0, x1;
      float a0[SPT][4], a1[SPT][4];
      load(x0, 0);
      float4 d0 = load_dt(0), d1 = load_dt(4);
      decays(a0, d0);
#pragma unroll 1
      for (int i = 0; i < S::TT; i += 16, pdt += 16, pdu += 16, pB += 16, pC += 16, py += 16) {
#pragma unroll
        for (int t = 0; t < 16; t += 8) {  // behind the tile's end: what is read there is not used
          load(x1, t + 4);
          d0 = load_dt(t + 8);
          decays(a1, d1);
          run(x0, a0, t);
          load(x0, t + 8);
          d1 = load_dt(t + 12);
          decays(a0, d0);
          run(x1, a1, t + 4);
        }
      }
    } else {  // no registers for a second set
#pragma unroll 1
      for (int i = 0; i < S::TT; i += 16, pdt += 16, pdu += 16, pB += 16, pC += 16, py += 16) {
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
          Operands x;
          float a[SPT][4];
          const float4 d = load_dt(t);
          load(x, t);
          decays(a, d);
          run(x, a, t);
        }
      }
    }
  }
};

template <typename T, bool WIDE, int RT, int SPT, int LP, int ST, int TT>
__global__ void __launch_bounds__(RT + 512, 1) selective_scan_kernel(const __grid_constant__ Maps maps, const lq_scan_problem p, bool by8) {
  using S = Shape<T, RT, SPT, LP, ST, TT>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  typename S::Smem& sm = *reinterpret_cast<typename S::Smem*>(smem_raw + ((128 - (smem_u32(smem_raw) & 127)) & 127));
  const int Dg = p.D / p.G, blocks = (Dg + S::CH - 1) / S::CH, row = blockIdx.x / blocks, b = row / p.G, grp = row - b * p.G;
  const int ch0 = ((int)blockIdx.x - row * blocks) * S::CH;  // within the group
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(smem_u32(&sm.full[i])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  pdl_enter();
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int tiles = (len + TT - 1) / TT;
  __syncthreads();
  // iteration i: the recurrence runs tile i, tile i + 1 is prepared, tile i - 1 is stored
  if (threadIdx.x < RT) {
    Recurrence<T, S, SPT, LP> r{sm, (int)threadIdx.x / LP, (int)threadIdx.x % LP};
    const bool on = ch0 + r.ch < Dg;
    const size_t at = (size_t)(grp * Dg + ch0 + r.ch) * p.N;
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
      const int n = r.ln + j * LP;
      const bool live = on && n < p.N;
      r.A[j] = live ? p.A[at + n] : 0.f;
      r.h[j] = live && p.initial_state ? p.initial_state[(size_t)b * p.D * p.N + at + n] : 0.f;
    }
    for (int i = -1; i <= tiles; ++i) {
      __syncthreads();
      if (i >= 0 && i < tiles) r.tile(i & 1);
    }
    if (p.final_state && on) {
      float* to = p.final_state + (size_t)b * p.D * p.N + at;
#pragma unroll
      for (int j = 0; j < SPT; ++j)
        if (r.ln + j * LP < p.N) to[r.ln + j * LP] = r.h[j];
    }
  } else if (threadIdx.x < RT + S::JOB) {
    Prepare<T, S, WIDE> job(p, maps, sm, (int)threadIdx.x - RT, b, grp, ch0, len);
    for (int i = -1; i <= tiles; ++i) {
      __syncthreads();
      if (i + 1 < tiles) job.run(i + 1);
    }
    if (!job.ok) {  // what was requested still lands
      for (int i = max(0, tiles - ST); i < tiles; ++i) mbar_wait_bounded(smem_u32(&sm.full[i % ST]), (uint32_t)((i / ST) & 1));
      if (p.status) atomicExch(p.status, 1);
    }
  } else {
    const Store<T, S, WIDE> job(by8, p, maps, sm, (int)threadIdx.x - RT - S::JOB, b, grp, ch0, len);
    for (int i = 0; i < ST - 2; ++i) job.request(i);
    job.arrived();
    for (int i = -1; i <= tiles; ++i) {
      __syncthreads();
      if (i > 0) {
        job.template run<LP>(i - 1);
        asm volatile("bar.sync 1, %0;\n" ::"n"(S::JOB) : "memory");  // nobody reads tile i - 1 any more
      }
      job.request(i + ST - 1);
      job.arrived();
    }
    cp_async_wait<0>();
    job.zeros(tiles * TT);
  }
}

static int encode(CUtensorMap* m, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return fail(LQ_ERR_LAUNCH, "selective_scan: the driver does not export cuTensorMapEncodeTiled");
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = dtype == LQ_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == LQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = enc(m, t, rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? LQ_OK : fail(LQ_ERR_LAUNCH, "selective_scan: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
}

template <typename T, int RT, int SPT, int LP, int ST, int TT>
static int launch_scan(const lq_scan_problem* p, cudaStream_t st) {
  using S = Shape<T, RT, SPT, LP, ST, TT>;
  const int Dg = p->D / p->G;
  constexpr int E = sizeof(T);
  const long long ctas = (long long)((Dg + S::CH - 1) / S::CH) * p->G * p->B;
  if (ctas >= (1ll << 31) - 1) return fail(LQ_ERR_SHAPE, "selective_scan: B=%d D=%d G=%d", p->B, p->D, p->G);
  // TMA: addresses, pitches and rows of 16 bytes; a pitch of 0 (an expanded input) is not one
  Maps maps = {};
  Alignment a;
  bool wide = S::CB % 16 == 0 && S::NB % 16 == 0 && p->T > 0;
  auto pitch = [&](long long elements, long long extent) {  // bytes; of no meaning where there is one
    if (extent == 1) return (cuuint64_t)16;
    a.pitch(elements, E);
    wide = wide && elements > 0;
    return (cuuint64_t)(elements * E);
  };
  struct In { CUtensorMap* map; const void* x; long long sb, st, sg; };
  const In in[5] = {{&maps.u, p->u, p->u_stride_b, p->u_stride_t, 0}, {&maps.dt, p->dt, p->dt_stride_b, p->dt_stride_t, 0},
                    {&maps.z, p->z, p->z_stride_b, p->z_stride_t, 0}, {&maps.B, p->Bm, p->B_stride_b, p->B_stride_t, p->B_stride_g},
                    {&maps.C, p->Cm, p->C_stride_b, p->C_stride_t, p->C_stride_g}};
  cuuint64_t pitches[5][3];
  for (int i = 0; i < 5; ++i) {
    if (in[i].x == nullptr) continue;
    a.at(in[i].x);
    pitches[i][0] = i < 3 ? 16 : pitch(in[i].sg, p->G);
    pitches[i][1] = pitch(in[i].st, p->T);
    pitches[i][2] = pitch(in[i].sb, p->B);
  }
  const bool by8 = Alignment(a).pitch(p->G > 1 ? Dg : 0, E).bytes() >= 8;
  wide = wide && a.at(p->y).pitch(Dg, E).pitch(p->N, E).bytes() == 16;
  for (int i = 0; i < 5 && wide; ++i) {
    if (in[i].x == nullptr) continue;
    const cuuint64_t chans[3] = {(cuuint64_t)p->D, (cuuint64_t)p->T, (cuuint64_t)p->B};
    const cuuint64_t states[4] = {(cuuint64_t)p->N, (cuuint64_t)p->G, (cuuint64_t)p->T, (cuuint64_t)p->B};
    const cuuint32_t cbox[3] = {S::CH, TT, 1}, nbox[4] = {S::NP, 1, TT, 1};
    if (int e = i < 3 ? encode(in[i].map, p->dtype, 3, in[i].x, chans, &pitches[i][1], cbox) : encode(in[i].map, p->dtype, 4, in[i].x, states, pitches[i], nbox)) return e;
  }
  auto go = [&](auto kern) { return launch_opt_in(kern, dim3((unsigned)ctas), dim3(S::THREADS), sizeof(typename S::Smem) + 128, st, maps, *p, by8); };
  const cudaError_t e = wide ? go(selective_scan_kernel<T, true, RT, SPT, LP, ST, TT>) : go(selective_scan_kernel<T, false, RT, SPT, LP, ST, TT>);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "selective_scan: %s", cudaGetErrorString(e));
  return check_launch("selective_scan_kernel");
}

// One CTA an SM. 16 channels a CTA leave each SM quadrant one warp of the recurrence, 64 channels two with twice the states: less
// time a channel where there are channels enough. Measured clocks a token and CTA (16 bits, gate): 44 against 128 with 16
// states, 42 against 94 with 8, 65 against 103 with 4; what counts is rounds of CTAs times that.
template <typename T>
static int run(const lq_scan_problem* p, cudaStream_t st) {
  constexpr int R = sizeof(T) == 2 ? 4 : 3, F = R + 1;  // tiles in the ring, as shared memory allows
  const long long sms = sm_count(), Dg = p->D / p->G, groups = (long long)p->B * p->G;
  auto narrow = [&](int clocks16, int clocks64) {
    const long long r16 = (groups * ((Dg + 15) / 16) + sms - 1) / sms, r64 = (groups * ((Dg + 63) / 64) + sms - 1) / sms;
    return r16 * clocks16 < r64 * clocks64;
  };
  if (p->N <= 4) return narrow(65, 103) ? launch_scan<T, 64, 1, 4, F, 64>(p, st) : launch_scan<T, 128, 2, 2, R, 32>(p, st);
  if (p->N <= 8) return narrow(42, 94) ? launch_scan<T, 64, 2, 4, F, 64>(p, st) : launch_scan<T, 128, 4, 2, R, 32>(p, st);
  if (p->N <= 16) return narrow(44, 128) ? launch_scan<T, 128, 2, 8, F, 64>(p, st) : launch_scan<T, 256, 4, 4, R, 32>(p, st);
  if (p->N <= 32) return launch_scan<T, 256, 4, 8, R, 32>(p, st);
  if (p->N <= 64) return launch_scan<T, 256, 4, 16, R, 32>(p, st);
  if (p->N <= 128) return launch_scan<T, 128, 8, 16, 3, 16>(p, st);
  return launch_scan<T, 128, 16, 16, 3, 16>(p, st);
}

// ------------------------------------------------------------------------------------------------ one token
// exp(dt A), as accurate as in the prompt's kernel: with fp32 inputs the rounding of a product with log2(e) would be the largest
// error of a step (60 ulps at dt A = -75)
template <typename T>
__device__ __forceinline__ float step_decay(float dt, float A) { return sizeof(T) == 4 ? expf(dt * A) : ex2(dt * kLog2e * A); }

// A row is the N states of one channel: lpr lanes hold it, VEC states each per step over N. HEADS: the channels of a head share a
// decay (heads whose channels are no multiple of four, states off 16 bytes or too many for one access of a warp).
template <typename T, typename TS, int VEC, bool HEADS>
__global__ void __launch_bounds__(128) selective_scan_step_kernel(const lq_scan_problem p, int lpr, bool wide_bc) {
  pdl_enter();
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const int ln = (int)(idx % lpr);
  const long long unit = idx / lpr;
  const bool live = unit < (long long)p.B * p.D;  // idle lanes still take part in the shuffles
  const int b = live ? (int)(unit / p.D) : 0, d = live ? (int)(unit - (long long)b * p.D) : 0;
  const int slot = p.slots ? p.slots[b] : b;
  const bool on = live && slot >= 0 && slot < p.n_slots;
  const int head = HEADS ? d / p.P : d;
  const int grp = HEADS ? head / (p.H / p.G) : d / (p.D / p.G);
  const T* Bm = reinterpret_cast<const T*>(p.Bm) + b * p.B_stride_b + grp * p.B_stride_g;
  const T* Cm = reinterpret_cast<const T*>(p.Cm) + b * p.C_stride_b + grp * p.C_stride_g;
  TS* state = reinterpret_cast<TS*>(p.state) + ((size_t)(on ? slot : 0) * p.D + d) * p.N;
  Pack<TS, VEC> raw;
  Pack<T, VEC> rB, rC;
  float A[HEADS ? 1 : VEC];
  auto request = [&](int n) {
    const bool in = on && n < p.N;
    raw.zero();
    rB.zero();
    rC.zero();
    if (in) {
      raw = load_pack<TS, VEC>(state + n);
      if (wide_bc) {
        rB = load_pack<T, VEC>(Bm + n);
        rC = load_pack<T, VEC>(Cm + n);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          rB.v[i] = Bm[n + i];
          rC.v[i] = Cm[n + i];
        }
      }
      if constexpr (!HEADS) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) A[i] = p.A[(size_t)d * p.N + n + i];
      }
    }
  };
  request(ln * VEC);  // the state first: everything else is small and comes out of the caches
  float dt = 0.f, u = 0.f, acc = 0.f;
  if (on) {
    dt = to_f32(reinterpret_cast<const T*>(p.dt)[b * p.dt_stride_b + head]) + (p.dt_bias ? p.dt_bias[head] : 0.f);
    if constexpr (HEADS) A[0] = p.A[head];
    u = to_f32(reinterpret_cast<const T*>(p.u)[b * p.u_stride_b + d]);
    dt = p.softplus ? softplus(dt) : dt;
    dt = clamp_nan(dt, p.dt_min, p.dt_max);
    const float head_decay = HEADS ? step_decay<T>(dt, A[0]) : 0.f, du = dt * u;
    for (int n = ln * VEC; n < p.N;) {
      float Bv[VEC], Cv[VEC], h[VEC];
      rB.get(Bv);
      rC.get(Cv);
      raw.get(h);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[i] = fmaf(HEADS ? head_decay : step_decay<T>(dt, A[HEADS ? 0 : i]), h[i], du * Bv[i]);
        acc = fmaf(h[i], Cv[i], acc);
      }
      raw.set(h);
      store_pack(state + n, raw);
      n += lpr * VEC;
      if (n < p.N) request(n);
    }
  }
  for (int m = lpr >> 1; m; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
  if (!live || ln != 0) return;
  if (p.skip) acc = fmaf(p.skip[HEADS && !p.skip_has_hdim ? head : d], u, acc);
  if (p.z && on) acc *= silu(to_f32(reinterpret_cast<const T*>(p.z)[b * p.z_stride_b + d]));
  reinterpret_cast<T*>(p.y)[(size_t)b * p.D + d] = from_f32<T>(on ? acc : 0.f);
}

// One decay a head and N states in one access of LPR lanes: a team walks over the channels of a head, R = 4 rows at a time, the
// next four requested while those at hand are stored (a load, its sum and its store one after the other reach 4.0 TB/s).
template <typename T, typename TS, int VEC>
__global__ void __launch_bounds__(128) heads_step_kernel(const lq_scan_problem p, int lpr, int groups, bool wide_bc) {
  pdl_enter();
  constexpr int R = 4;
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const int ln = (int)(idx % lpr), per_head = p.P / (R * groups);
  const long long unit = idx / lpr;
  const bool live = unit < (long long)p.B * p.H * per_head;  // idle lanes still take part in the shuffles
  const int b = live ? (int)(unit / (p.H * per_head)) : 0, in_b = live ? (int)(unit - (long long)b * p.H * per_head) : 0;
  const int head = in_b / per_head, d0 = head * p.P + (in_b - head * per_head) * R * groups, grp = head / (p.H / p.G), n = ln * VEC;
  const int slot = p.slots ? p.slots[b] : b;
  const bool on = live && slot >= 0 && slot < p.n_slots, in = on && n < p.N;
  TS* state = reinterpret_cast<TS*>(p.state) + ((size_t)(on ? slot : 0) * p.D + d0) * p.N + n;
  const T* u = reinterpret_cast<const T*>(p.u) + b * p.u_stride_b + d0;
  Pack<TS, VEC> next[R];
  T nu[R];
  auto request = [&](int g) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (in) next[r] = load_pack<TS, VEC>(state + (size_t)(g * R + r) * p.N);
      else next[r].zero();
      nu[r] = on ? u[g * R + r] : from_f32<T>(0.f);
    }
  };
  request(0);
  float Bv[VEC], Cv[VEC];
  {
    Pack<T, VEC> rB, rC;
    rB.zero();
    rC.zero();
    const T* Bm = reinterpret_cast<const T*>(p.Bm) + b * p.B_stride_b + grp * p.B_stride_g + n;
    const T* Cm = reinterpret_cast<const T*>(p.Cm) + b * p.C_stride_b + grp * p.C_stride_g + n;
    if (in && wide_bc) {
      rB = load_pack<T, VEC>(Bm);
      rC = load_pack<T, VEC>(Cm);
    } else if (in) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        rB.v[i] = Bm[i];
        rC.v[i] = Cm[i];
      }
    }
    rB.get(Bv);
    rC.get(Cv);
  }
  float decay = 0.f;
  if (on) {
    float dt = to_f32(reinterpret_cast<const T*>(p.dt)[b * p.dt_stride_b + head]) + (p.dt_bias ? p.dt_bias[head] : 0.f);
    dt = clamp_nan(p.softplus ? softplus(dt) : dt, p.dt_min, p.dt_max);
    decay = step_decay<T>(dt, p.A[head]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) Bv[i] *= dt;
  }
  for (int g = 0; g < groups; ++g) {
    Pack<TS, VEC> raw[R];
    float uu[R], acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      raw[r] = next[r];
      uu[r] = to_f32(nu[r]);
    }
    if (g + 1 < groups) request(g + 1);
    const int d = d0 + g * R;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float h[VEC];
      raw[r].get(h);
      acc[r] = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[i] = fmaf(decay, h[i], uu[r] * Bv[i]);
        acc[r] = fmaf(h[i], Cv[i], acc[r]);
      }
      raw[r].set(h);
      if (in) store_pack(state + (size_t)(g * R + r) * p.N, raw[r]);
    }
    int row;
    if (lpr >= 4) {  // rows are handed out over the lanes while they are summed: each lane ends with one row
      const bool hi = ln & (lpr >> 1), hi2 = ln & (lpr >> 2);
      float a0 = hi ? acc[2] : acc[0], a1 = hi ? acc[3] : acc[1];
      a0 += __shfl_xor_sync(0xffffffffu, hi ? acc[0] : acc[2], lpr >> 1);
      a1 += __shfl_xor_sync(0xffffffffu, hi ? acc[1] : acc[3], lpr >> 1);
      float v = hi2 ? a1 : a0;
      v += __shfl_xor_sync(0xffffffffu, hi2 ? a0 : a1, lpr >> 2);
      for (int m = lpr >> 3; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
      acc[0] = v;
      row = 2 * hi + hi2;
      if (ln & ((lpr >> 2) - 1)) row = R;  // one lane of each row's writes it
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        for (int m = lpr >> 1; m; m >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], m);
      row = -1;  // lane 0 writes all
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!live || !(row == r || (row == -1 && ln == 0))) continue;
      float v = row < 0 ? acc[r] : acc[0];
      if (p.skip) v = fmaf(p.skip[p.skip_has_hdim ? d + r : head], uu[r], v);
      if (p.z && on) v *= silu(to_f32(reinterpret_cast<const T*>(p.z)[b * p.z_stride_b + d + r]));
      reinterpret_cast<T*>(p.y)[(size_t)b * p.D + d + r] = from_f32<T>(on ? v : 0.f);
    }
  }
}
template <typename T, typename TS, int VEC>
static int launch_heads(const lq_scan_problem* p, cudaStream_t st) {
  int lpr = 1, groups = p->P / 4;
  while (lpr * VEC < p->N) lpr *= 2;
  // as many channels a team as leave threads for the GPU
  auto threads = [&] { return (long long)p->B * p->H * (p->P / (4 * groups)) * lpr; };
  while (groups > 1 && groups % 2 == 0 && threads() < (long long)sm_count() * 1024) groups /= 2;
  if (threads() == 0) return LQ_OK;
  if (threads() / 128 >= (1ll << 31) - 1) return fail(LQ_ERR_SHAPE, "selective_scan_step: B=%d D=%d N=%d", p->B, p->D, p->N);
  constexpr int E = sizeof(T), BYTES = VEC * E < 16 ? VEC * E : 16;
  Alignment a;
  a.at(p->Bm).at(p->Cm).pitch(p->B_stride_b, E).pitch(p->B_stride_g, E).pitch(p->C_stride_b, E).pitch(p->C_stride_g, E);
  launch(heads_step_kernel<T, TS, VEC>, dim3((unsigned)((threads() + 127) / 128)), dim3(128), 0, st, *p, lpr, groups, a.bytes() >= BYTES);
  return check_launch("heads_step_kernel");
}

template <typename T, typename TS, int VEC, bool HEADS>
static int launch_step(const lq_scan_problem* p, cudaStream_t st) {
  int lpr = 1;
  while (lpr < 32 && lpr * VEC < p->N) lpr *= 2;
  const long long threads = (long long)p->B * p->D * lpr;
  if (threads == 0) return LQ_OK;
  if (threads / 128 >= (1ll << 31) - 1) return fail(LQ_ERR_SHAPE, "selective_scan_step: B=%d D=%d N=%d", p->B, p->D, p->N);
  constexpr int E = sizeof(T), BYTES = VEC * E < 16 ? VEC * E : 16;
  Alignment a;
  a.at(p->Bm).at(p->Cm).pitch(p->B_stride_b, E).pitch(p->B_stride_g, E).pitch(p->C_stride_b, E).pitch(p->C_stride_g, E);
  launch(selective_scan_step_kernel<T, TS, VEC, HEADS>, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, st, *p, lpr, a.bytes() >= BYTES);
  return check_launch("selective_scan_step_kernel");
}
template <typename T, typename TS>
static int run_step(const lq_scan_problem* p, cudaStream_t st) {
  constexpr int FULL = 16 / sizeof(TS);
  Alignment a;
  const bool wide = a.at(p->state).pitch(p->N, sizeof(TS)).bytes() == 16;
  if (p->H == 0) return wide ? launch_step<T, TS, FULL, false>(p, st) : launch_step<T, TS, 1, false>(p, st);
  if (p->P % 4 == 0 && wide && p->N <= 32 * FULL) return launch_heads<T, TS, FULL>(p, st);
  return wide ? launch_step<T, TS, FULL, true>(p, st) : launch_step<T, TS, 1, true>(p, st);
}

static int check(const lq_scan_problem* p, bool step, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->B < 0 || p->T < 0 || p->D <= 0 || p->G <= 0 || p->N <= 0 || p->D % p->G || !fits(p->T) || !fits(p->D))
    return fail(LQ_ERR_SHAPE, "%s: B=%d T=%d D=%d N=%d G=%d", what, p->B, p->T, p->D, p->N, p->G);
  if (p->N > 256) return fail(LQ_ERR_UNSUPPORTED, "%s: %d states a channel (at most 256)", what, p->N);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d", what, p->dtype);
  if (!p->A || ((!p->u || !p->dt || !p->Bm || !p->Cm || !p->y) && (long long)p->B * p->T > 0))
    return fail(LQ_ERR_NULL, "%s: u, dt, A, B, C and y must be non-null", what);
  if (!step) return p->H ? fail(LQ_ERR_UNSUPPORTED, "%s: one decay rate a head is for single tokens", what) : LQ_OK;
  if (p->T != 1) return fail(LQ_ERR_SHAPE, "%s: T=%d, one token expected", what, p->T);
  if (p->H && (p->P <= 0 || (long long)p->H * p->P != p->D || p->H % p->G)) return fail(LQ_ERR_SHAPE, "%s: H=%d P=%d D=%d G=%d", what, p->H, p->P, p->D, p->G);
  if (p->state_dtype < LQ_F16 || p->state_dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "%s: state dtype %d", what, p->state_dtype);
  if (!p->state) return fail(LQ_ERR_NULL, "%s: state is null", what);
  if (!p->slots && p->n_slots < p->B) return fail(LQ_ERR_SHAPE, "%s: %d slots for %d sequences", what, p->n_slots, p->B);
  return LQ_OK;
}

}  // namespace scan
}  // namespace lq

extern "C" int lq_selective_scan_fwd(const lq_scan_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = scan::check(p, false, "selective_scan")) return e;
  if (p->B == 0) return LQ_OK;
  return with_dtype(p->dtype, "selective_scan", [&](auto t) { return scan::run<decltype(t)>(p, (cudaStream_t)stream); });
}

extern "C" int lq_selective_scan_step(const lq_scan_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = scan::check(p, true, "selective_scan_step")) return e;
  return with_dtype(p->dtype, "selective_scan_step", [&](auto t) {
    return with_dtype(p->state_dtype, "selective_scan_step", [&](auto s) { return scan::run_step<decltype(t), decltype(s)>(p, (cudaStream_t)stream); });
  });
}
