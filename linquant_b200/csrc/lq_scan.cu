// Selective scan over the tokens of a prompt, one decay rate per channel and state.
//
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n],   y_t = sum_n C_t[n] h_t[n] + skip u_t,   y_t *= silu(z_t)
//
// Bound by the exponentials: one per token, channel and state at 16 a clock and SM. A channel's states are spread over LP
// lanes with SPT states in the registers of each, so every exponential is computed once and no lane recomputes another's
// part; tokens go one after the other, a tile of them at a time through shared memory (dt and dt u of the tile's channels,
// B and C shared by the channels of a group), and a lane's part of y_t is summed over the LP lanes when the tile is stored.
#include "lq_layer.cuh"

namespace lq {

namespace scan {

template <typename T, int SPT, int LP, int THREADS, int TT>
struct Shape {
  static constexpr int NP = SPT * LP, CH = THREADS / LP, EPT = TT > LP ? TT / LP : 1;  // EPT: elements of a tile a thread loads and stores
  struct Smem {
    float2 step[TT][CH];  // dt, dt u
    float y[TT][THREADS];
    float B[TT][NP], C[TT][NP];
  };
};

template <typename T, int SPT, int LP, int THREADS, int TT>
__global__ void __launch_bounds__(THREADS) selective_scan_kernel(const lq_scan_problem p) {
  pdl_enter();
  using S = Shape<T, SPT, LP, THREADS, TT>;
  constexpr int NP = S::NP, CH = S::CH, EPT = S::EPT;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  typename S::Smem& sm = *reinterpret_cast<typename S::Smem*>(smem_raw);
  const int tid = threadIdx.x, b = blockIdx.z, grp = blockIdx.y, Dg = p.D / p.G;
  const int ch0 = blockIdx.x * CH;                    // within the group
  const int ch = tid / LP, ln = tid % LP;             // recurrence: channel and first state / SPT of this thread
  const int ech = tid % CH, et = tid / CH;            // loads and stores: channel and first token
  const bool on = ch0 + ch < Dg, eon = ch0 + ech < Dg;
  const int d = grp * Dg + ch0 + ch, ed = grp * Dg + ch0 + ech;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;

  float a2[SPT], h[SPT];
#pragma unroll
  for (int j = 0; j < SPT; ++j) {
    const int n = ln * SPT + j;
    const bool live = on && n < p.N;
    a2[j] = live ? p.A[(size_t)d * p.N + n] * kLog2e : 0.f;
    h[j] = live && p.initial_state ? p.initial_state[((size_t)b * p.D + d) * p.N + n] : 0.f;
  }
  const float bias = eon && p.dt_bias ? p.dt_bias[ed] : 0.f, skip = eon && p.skip ? p.skip[ed] : 0.f;
  const T* u = reinterpret_cast<const T*>(p.u) + b * p.u_stride_b + ed;
  const T* dt = reinterpret_cast<const T*>(p.dt) + b * p.dt_stride_b + ed;
  const T* z = p.z ? reinterpret_cast<const T*>(p.z) + b * p.z_stride_b + ed : nullptr;
  const T* Bm = reinterpret_cast<const T*>(p.Bm) + b * p.B_stride_b + grp * p.B_stride_g;
  const T* Cm = reinterpret_cast<const T*>(p.Cm) + b * p.C_stride_b + grp * p.C_stride_g;
  T* y = reinterpret_cast<T*>(p.y) + (size_t)b * p.T * p.D + ed;
  constexpr int ESTEP = LP;  // tokens between a thread's elements
  const bool ein = et < TT;

  for (int t0 = 0; t0 < len; t0 += TT) {
    float uu[EPT], zz[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int t = t0 + et + i * ESTEP;
      const bool live = eon && t < len;
      uu[i] = live ? to_f32(u[t * p.u_stride_t]) : 0.f;
      zz[i] = live && z ? to_f32(z[t * p.z_stride_t]) : 0.f;
      float v = live ? to_f32(dt[t * p.dt_stride_t]) + bias : 0.f;
      v = p.softplus ? softplus(v) : v;
      v = clamp_nan(v, p.dt_min, p.dt_max);
      if (ein) sm.step[et + i * ESTEP][ech] = live ? make_float2(v, v * uu[i]) : make_float2(0.f, 0.f);
    }
    for (int i = tid; i < TT * NP; i += THREADS) {
      const int tt = i / NP, n = i % NP, t = t0 + tt;
      const bool live = t < len && n < p.N;  // what lies behind the last token takes no part, not even as 0 x NaN
      sm.B[tt][n] = live ? to_f32(Bm[t * p.B_stride_t + n]) : 0.f;
      sm.C[tt][n] = live ? to_f32(Cm[t * p.C_stride_t + n]) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int tt = 0; tt < TT; ++tt) {
      const float2 s = sm.step[tt][ch];
      float acc = 0.f;
#pragma unroll
      for (int j = 0; j < SPT; ++j) {
        h[j] = fmaf(ex2(s.x * a2[j]), h[j], s.y * sm.B[tt][ln * SPT + j]);
        acc = fmaf(h[j], sm.C[tt][ln * SPT + j], acc);
      }
      sm.y[tt][tid] = acc;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int tt = et + i * ESTEP, t = t0 + tt;
      if (!ein) break;
      float v = skip * uu[i];
#pragma unroll
      for (int l = 0; l < LP; ++l) v += sm.y[tt][ech * LP + l];
      if (z) v *= silu(zz[i]);
      if (eon && t < p.T) y[(size_t)t * p.D] = from_f32<T>(t < len ? v : 0.f);
    }
  }
  if (eon && ein)  // tiles that no token reaches
    for (int t = (len + TT - 1) / TT * TT + et; t < p.T; t += ESTEP < TT ? ESTEP : TT) y[(size_t)t * p.D] = from_f32<T>(0.f);
  if (p.final_state && on) {
#pragma unroll
    for (int j = 0; j < SPT; ++j)
      if (ln * SPT + j < p.N) p.final_state[((size_t)b * p.D + d) * p.N + ln * SPT + j] = h[j];
  }
}

template <typename T, int SPT, int LP>
static int launch_scan(const lq_scan_problem* p, cudaStream_t st) {
  constexpr int THREADS = 256, TT = SPT * LP > 64 ? 16 : 32;
  using S = Shape<T, SPT, LP, THREADS, TT>;
  const int Dg = p->D / p->G;
  const dim3 grid((Dg + S::CH - 1) / S::CH, p->G, p->B);
  if (grid.y > 65535 || grid.z > 65535) return fail(LQ_ERR_SHAPE, "selective_scan: B=%d G=%d", p->B, p->G);
  const cudaError_t e = launch_opt_in(selective_scan_kernel<T, SPT, LP, THREADS, TT>, grid, dim3(THREADS), sizeof(typename S::Smem), st, *p);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "selective_scan: %s", cudaGetErrorString(e));
  return check_launch("selective_scan_kernel");
}

template <typename T>
static int run(const lq_scan_problem* p, cudaStream_t st) {
  if (p->N <= 4) return launch_scan<T, 4, 1>(p, st);
  if (p->N <= 8) return launch_scan<T, 4, 2>(p, st);
  if (p->N <= 16) return launch_scan<T, 4, 4>(p, st);
  if (p->N <= 32) return launch_scan<T, 4, 8>(p, st);
  if (p->N <= 64) return launch_scan<T, 4, 16>(p, st);
  if (p->N <= 128) return launch_scan<T, 4, 32>(p, st);
  return launch_scan<T, 8, 32>(p, st);
}

// ------------------------------------------------------------------------------------------------ one token
// A row is the N states of one channel. LPR lanes hold it, VEC states each per step over N; a thread group takes R rows of
// one head (HEADS: they share the decay, B and C) or one row with a decay rate per state.
template <typename T, typename TS, int VEC, int R, bool HEADS>
__global__ void __launch_bounds__(128) selective_scan_step_kernel(const lq_scan_problem p, int lpr) {
  pdl_enter();
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const int ln = (int)(idx % lpr), per_b = p.D / R;
  const long long unit = idx / lpr;
  const bool live = unit < (long long)p.B * per_b;  // idle lanes still take part in the shuffles
  const int b = live ? (int)(unit / per_b) : 0, d0 = live ? (int)(unit - (long long)b * per_b) * R : 0;
  const int slot = p.slots ? p.slots[b] : b;
  const bool on = live && slot >= 0 && slot < p.n_slots;
  const int head = HEADS ? d0 / p.P : d0;
  const int grp = HEADS ? head / (p.H / p.G) : d0 / (p.D / p.G);
  float dt = 0.f;
  if (on) {
    dt = to_f32(reinterpret_cast<const T*>(p.dt)[b * p.dt_stride_b + head]) + (p.dt_bias ? p.dt_bias[head] : 0.f);
    dt = p.softplus ? softplus(dt) : dt;
    dt = clamp_nan(dt, p.dt_min, p.dt_max);
  }
  const T* Bm = reinterpret_cast<const T*>(p.Bm) + b * p.B_stride_b + grp * p.B_stride_g;
  const T* Cm = reinterpret_cast<const T*>(p.Cm) + b * p.C_stride_b + grp * p.C_stride_g;
  float u[R], acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    u[r] = on ? to_f32(reinterpret_cast<const T*>(p.u)[b * p.u_stride_b + d0 + r]) : 0.f;
    acc[r] = 0.f;
  }
  const float head_decay = HEADS && on ? ex2(dt * (p.A[head] * kLog2e)) : 0.f;
  if (on) {
    TS* state = reinterpret_cast<TS*>(p.state) + ((size_t)slot * p.D + d0) * p.N;
    for (int n = ln * VEC; n < p.N; n += lpr * VEC) {
      Pack<TS, VEC> raw[R];
#pragma unroll
      for (int r = 0; r < R; ++r) raw[r] = load_pack<TS, VEC>(state + (size_t)r * p.N + n);
      float Bv[VEC], Cv[VEC], a[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        Bv[i] = to_f32(Bm[n + i]);
        Cv[i] = to_f32(Cm[n + i]);
        a[i] = HEADS ? head_decay : ex2(dt * (p.A[(size_t)d0 * p.N + n + i] * kLog2e));
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float h[VEC];
        raw[r].get(h);
        const float du = dt * u[r];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          h[i] = fmaf(a[i], h[i], du * Bv[i]);
          acc[r] = fmaf(h[i], Cv[i], acc[r]);
        }
        raw[r].set(h);
        store_pack(state + (size_t)r * p.N + n, raw[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    for (int m = lpr >> 1; m; m >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], m);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!live || ln != r % lpr) continue;
    const int d = d0 + r;
    float v = acc[r];
    if (p.skip) v = fmaf(p.skip[HEADS && !p.skip_has_hdim ? head : d], u[r], v);
    if (p.z && on) v *= silu(to_f32(reinterpret_cast<const T*>(p.z)[b * p.z_stride_b + d]));
    reinterpret_cast<T*>(p.y)[(size_t)b * p.D + d] = from_f32<T>(on ? v : 0.f);
  }
}

template <typename T, typename TS, int VEC, int R, bool HEADS>
static int launch_step(const lq_scan_problem* p, cudaStream_t st) {
  int lpr = 1;
  while (lpr < 32 && lpr * VEC < p->N) lpr *= 2;
  const long long threads = (long long)p->B * (p->D / R) * lpr;
  if (threads == 0) return LQ_OK;
  if (threads / 128 >= (1ll << 31) - 1) return fail(LQ_ERR_SHAPE, "selective_scan_step: B=%d D=%d N=%d", p->B, p->D, p->N);
  launch(selective_scan_step_kernel<T, TS, VEC, R, HEADS>, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, st, *p, lpr);
  return check_launch("selective_scan_step_kernel");
}
template <typename T, typename TS>
static int run_step(const lq_scan_problem* p, cudaStream_t st) {
  constexpr int FULL = 16 / sizeof(TS);
  Alignment a;
  const bool wide = a.at(p->state).pitch(p->N, sizeof(TS)).bytes() == 16;
  if (p->H == 0) return wide ? launch_step<T, TS, FULL, 1, false>(p, st) : launch_step<T, TS, 1, 1, false>(p, st);
  if (p->P % 4 == 0) return wide ? launch_step<T, TS, FULL, 4, true>(p, st) : launch_step<T, TS, 1, 4, true>(p, st);
  return wide ? launch_step<T, TS, FULL, 1, true>(p, st) : launch_step<T, TS, 1, 1, true>(p, st);
}

static int check(const lq_scan_problem* p, bool step, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->B < 0 || p->T < 0 || p->D <= 0 || p->G <= 0 || p->N <= 0 || p->D % p->G)
    return fail(LQ_ERR_SHAPE, "%s: B=%d T=%d D=%d N=%d G=%d", what, p->B, p->T, p->D, p->N, p->G);
  if (p->N > 256) return fail(LQ_ERR_UNSUPPORTED, "%s: %d states a channel (at most 256)", what, p->N);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d", what, p->dtype);
  if (!p->A || ((!p->u || !p->dt || !p->Bm || !p->Cm || !p->y) && (long long)p->B * p->T > 0))
    return fail(LQ_ERR_NULL, "%s: u, dt, A, B, C and y must be non-null", what);
  if (!step) return p->H ? fail(LQ_ERR_UNSUPPORTED, "%s: one decay rate a head is for single tokens", what) : LQ_OK;
  if (p->T != 1) return fail(LQ_ERR_SHAPE, "%s: T=%d, one token expected", what, p->T);
  if (p->H && (p->P <= 0 || p->H * p->P != p->D || p->H % p->G)) return fail(LQ_ERR_SHAPE, "%s: H=%d P=%d D=%d G=%d", what, p->H, p->P, p->D, p->G);
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
