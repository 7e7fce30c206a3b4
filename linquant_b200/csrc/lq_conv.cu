// Short causal convolution over the tokens of each channel, with its activation: prompts and single tokens.
//
//   y[t] = act( bias + sum_{i < W} w[i] x[t - W + 1 + i] )          x before the first token from the cached state
//
// Memory-bound: x is read once and y written once, 2 W flops and one SiLU a value.
#include "lq_layer.cuh"

namespace lq {

namespace conv {

template <typename T, int W, int VEC>
struct Taps {
  float w[VEC][W], b[VEC];
  __device__ __forceinline__ Taps(const lq_conv_problem& p, int c) {
    // the taps of a thread's channels lie one after the other: pieces as large as the channels' alignment allows
    constexpr int PIECE = VEC * W % 4 == 0 ? 4 : VEC * W % 2 == 0 ? 2 : 1;
    const float* from = p.weight + (size_t)c * W;
    if ((reinterpret_cast<uintptr_t>(from) & (4 * PIECE - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < VEC * W; i += PIECE) {
        const Pack<float, PIECE> v = load_pack<float, PIECE>(from + i);
#pragma unroll
        for (int k = 0; k < PIECE; ++k) w[(i + k) / W][(i + k) % W] = v.v[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC * W; ++i) w[i / W][i % W] = __ldg(from + i);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) b[i] = p.bias ? __ldg(p.bias + c + i) : 0.f;
  }
  // line: the W inputs of a token, oldest first
  __device__ __forceinline__ Pack<T, VEC> out(const float (&line)[W][VEC], bool act) const {
    float y[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float s = b[i];
#pragma unroll
      for (int k = 0; k < W; ++k) s = fmaf(line[k][i], w[i][k], s);
      y[i] = act ? silu(s) : s;
    }
    Pack<T, VEC> r;
    r.set(y);
    return r;
  }
};

// A thread walks a run of tokens of VEC channels with the last W-1 inputs in registers;
// the threads behind the last run write the final state.
template <typename T, int W, int VEC, bool ACT>
__global__ void __launch_bounds__(128) short_conv_kernel(const lq_conv_problem p, int run, int runs) {
  pdl_enter();
  constexpr bool WIDE = VEC * sizeof(T) == 16;
  constexpr int U = WIDE ? 4 : 8, RING = 16;
  __shared__ Pack<T, VEC> ring[WIDE ? RING : 1][WIDE ? 128 : 1];
  const int nvec = p.D / VEC, per_b = runs + (p.final_state != nullptr);
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const long long rest = idx / nvec;
  const int c = (int)(idx - rest * nvec) * VEC, b = (int)(rest / per_b), seg = (int)(rest - (long long)b * per_b);
  if (b >= p.B) return;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + c;
  const T* before = p.initial_state ? reinterpret_cast<const T*>(p.initial_state) + (size_t)b * (W - 1) * p.D + c : nullptr;
  auto input = [&](int t) {  // t < n; negative: ahead of the first token
    Pack<T, VEC> v;
    if (t >= 0) v = load_pack<T, VEC>(x + t * p.x_stride_t);
    else if (before) v = load_pack<T, VEC>(before + (size_t)(W - 1 + t) * p.D);
    else v.zero();
    return v;
  };
  if (seg == runs) {
    T* fs = reinterpret_cast<T*>(p.final_state) + (size_t)b * (W - 1) * p.D + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_pack(fs + (size_t)j * p.D, input(n - (W - 1) + j));
    return;
  }
  const int t0 = seg * run, t1 = min(t0 + run, p.T), live = min(t1, n);
  T* y = reinterpret_cast<T*>(p.y) + (size_t)b * p.T * p.D + c;
  if (t0 < live) {
    const Taps<T, W, VEC> taps(p, c);
    float line[W][VEC];
#pragma unroll
    for (int k = 1; k < W; ++k) input(t0 - W + k).get(line[k]);
    T* to = y + (size_t)t0 * p.D;
    auto next = [&](const Pack<T, VEC>& raw) {
#pragma unroll
      for (int k = 0; k + 1 < W; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) line[k][i] = line[k + 1][i];
      raw.get(line[W - 1]);
      store_pack(to, taps.out(line, ACT));
      to += p.D;
    };
    const T* from = x + t0 * p.x_stride_t;
    if constexpr (VEC * sizeof(T) == 16) {  // tokens arrive in a ring of the thread's own: AHEAD of them on their way without registers
      auto issue = [&](int g) {
#pragma unroll
        for (int u = 0; u < U; ++u, from += p.x_stride_t)
          if (t0 + g * U + u < live) cp_async16(&ring[(g * U + u) % RING][threadIdx.x], from);
        cp_async_commit();
      };
#pragma unroll
      for (int g = 0; g < RING / U - 1; ++g) issue(g);
      for (int g = 0, t = t0; t < live; ++g, t += U) {
        issue(g + RING / U - 1);
        cp_async_wait<RING / U - 1>();
        if (t + U <= live) {
#pragma unroll
          for (int u = 0; u < U; ++u) next(ring[(g * U + u) % RING][threadIdx.x]);
        } else {
          for (int u = 0; t + u < live; ++u) next(ring[(g * U + u) % RING][threadIdx.x]);
        }
      }
      cp_async_wait<0>();
    } else {
      int t = t0;
      for (; t + U <= live; t += U) {
        Pack<T, VEC> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u, from += p.x_stride_t) raw[u] = load_pack<T, VEC>(from);
#pragma unroll
        for (int u = 0; u < U; ++u) next(raw[u]);
      }
#pragma unroll 1
      for (; t < live; ++t, from += p.x_stride_t) next(load_pack<T, VEC>(from));
    }
  }
  Pack<T, VEC> none;
  none.zero();
  for (int t = max(t0, live); t < t1; ++t) store_pack(y + (size_t)t * p.D, none);
}

template <typename T, int W, int VEC>
__global__ void __launch_bounds__(128) short_conv_step_kernel(const lq_conv_problem p) {
  pdl_enter();
  const int nvec = p.D / VEC;
  const long long idx = (long long)blockIdx.x * 128 + threadIdx.x;
  const int b = (int)(idx / nvec), c = (int)(idx - (long long)b * nvec) * VEC;
  if (b >= p.B) return;
  const int slot = p.slots ? p.slots[b] : b;
  const Taps<T, W, VEC> taps(p, c);
  Pack<T, VEC> raw[W];
  raw[W - 1] = load_pack<T, VEC>(reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + c);
  T* y = reinterpret_cast<T*>(p.y) + (size_t)b * p.D + c;
  if (slot < 0 || slot >= p.n_slots) {
    Pack<T, VEC> none;
    none.zero();
    store_pack(y, none);
    return;
  }
  T* state = reinterpret_cast<T*>(p.state) + (size_t)slot * (W - 1) * p.D + c;
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) raw[k] = load_pack<T, VEC>(state + (size_t)k * p.D);
  float line[W][VEC];
#pragma unroll
  for (int k = 0; k < W; ++k) raw[k].get(line[k]);
  store_pack(y, taps.out(line, p.silu));
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) store_pack(state + (size_t)k * p.D, raw[k + 1]);
}

static int check(const lq_conv_problem* p, bool step, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->B < 0 || p->T < 0 || p->D <= 0 || !fits(p->T) || !fits(p->D)) return fail(LQ_ERR_SHAPE, "%s: B=%d T=%d D=%d", what, p->B, p->T, p->D);
  if (p->W < 2 || p->W > 4) return fail(LQ_ERR_UNSUPPORTED, "%s: %d taps (2, 3 or 4)", what, p->W);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d", what, p->dtype);
  if (!p->weight || ((!p->x || !p->y) && (long long)p->B * p->T > 0)) return fail(LQ_ERR_NULL, "%s: x, weight and y must be non-null", what);
  if (step && p->T != 1) return fail(LQ_ERR_SHAPE, "%s: T=%d, one token expected", what, p->T);
  if (step && !p->state) return fail(LQ_ERR_NULL, "%s: state is null", what);
  if (step && !p->slots && p->n_slots < p->B) return fail(LQ_ERR_SHAPE, "%s: %d slots for %d sequences", what, p->n_slots, p->B);
  return LQ_OK;
}
template <typename F>
static int with_taps(int W, F&& f) {
  return W == 2 ? f(std::integral_constant<int, 2>()) : W == 3 ? f(std::integral_constant<int, 3>()) : f(std::integral_constant<int, 4>());
}

template <typename T, int VEC>
static int run_fwd(const lq_conv_problem* p, cudaStream_t st) {
  // Long runs load the taps and the inputs ahead of a run (W - 1) less often, short ones fill the GPU
  const long long lanes = (long long)p->B * (p->D / VEC), fill = (long long)sm_count() * 512;
  const int run = lanes * (p->T / 128) >= 3 * fill ? 128 : lanes * (p->T / 32) >= fill ? 32 : 8;
  const int runs = (p->T + run - 1) / run;
  const long long threads = lanes * (runs + (p->final_state != nullptr));
  if (threads == 0) return LQ_OK;
  if (threads / 128 >= (1ll << 31) - 1) return fail(LQ_ERR_SHAPE, "short_conv: B=%d T=%d D=%d", p->B, p->T, p->D);
  return with_taps(p->W, [&](auto w) {
    auto go = [&](auto kern) { launch(kern, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, st, *p, run, runs); };
    if (p->silu) go(short_conv_kernel<T, decltype(w)::value, VEC, true>);
    else go(short_conv_kernel<T, decltype(w)::value, VEC, false>);
    return check_launch("short_conv_kernel");
  });
}
template <typename T, int VEC>
static int run_step(const lq_conv_problem* p, cudaStream_t st) {
  const long long threads = (long long)p->B * (p->D / VEC);
  if (threads == 0) return LQ_OK;
  return with_taps(p->W, [&](auto w) {
    launch(short_conv_step_kernel<T, decltype(w)::value, VEC>, dim3((unsigned)((threads + 127) / 128)), dim3(128), 0, st, *p);
    return check_launch("short_conv_step_kernel");
  });
}

}  // namespace conv
}  // namespace lq

extern "C" int lq_short_conv_fwd(const lq_conv_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = conv::check(p, false, "short_conv")) return e;
  return with_dtype(p->dtype, "short_conv", [&](auto t) {
    using T = decltype(t);
    constexpr int FULL = 16 / sizeof(T);
    Alignment a;
    a.at(p->x).at(p->y).at(p->initial_state).at(p->final_state).pitch(p->x_stride_b, sizeof(T)).pitch(p->x_stride_t, sizeof(T)).pitch(p->D, sizeof(T));
    return a.bytes() == 16 ? conv::run_fwd<T, FULL>(p, (cudaStream_t)stream) : conv::run_fwd<T, 1>(p, (cudaStream_t)stream);
  });
}

extern "C" int lq_short_conv_step(const lq_conv_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = conv::check(p, true, "short_conv_step")) return e;
  return with_dtype(p->dtype, "short_conv_step", [&](auto t) {
    using T = decltype(t);
    Alignment a;  // two channels a thread: more of them share the latency of the loads
    a.at(p->x).at(p->y).at(p->state).pitch(p->x_stride_b, sizeof(T)).pitch(p->D, sizeof(T));
    return a.bytes() >= 2 * (int)sizeof(T) ? conv::run_step<T, 2>(p, (cudaStream_t)stream) : conv::run_step<T, 1>(p, (cudaStream_t)stream);
  });
}
