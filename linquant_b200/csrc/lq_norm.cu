// Norms around a block, and the row quantiser of the INT8 products.
//
//   lq_rms_norm         r = residual + alpha P(x),  P(x) = x or norm(x) post_weight;   y = norm(r) weight
//   lq_gated_rms_norm   y = norm(x silu(gate)) weight,  or  norm(x) weight silu(gate)
//   lq_quantize_rows    y = x
//   norm(v) = v / sqrt(mean(v^2) + eps) over a row (or over each group of its channels); y leaves as f16 / bf16 / f32 or as
//   INT8 codes with one scale a row (amax / 127).
//
// Memory-bound: every input is read once into registers (VEC values a load, NV loads a thread), the sums of a row are taken
// in fp32 by the team of threads that holds it, and y, r and the codes are written once: gated norm of 32768 x 5120 bf16 186 us
// (5.4 TB/s; 213 with INT8 outputs, 3.9), residual and norm of 16384 x 2560 56.6 us (5.9).
// Rows off a pack's boundary are walked in packs too where all tensors lie at the same distance behind theirs. Where they do not (an odd
// row length next to a slice, to an fp32 residual or to another output type; groups that are no multiple of a pack) a value goes by
// itself and rows of more than 1024 spill: gated norm of 32768 x 2561 153 us against 756 with the gate a slice.
#include "lq_layer.cuh"

namespace lq {

namespace norm {

constexpr int MOST = 16384;  // channels that are normed together

enum Kind { PLAIN, ADD, ADD32, GATED };  // ADD32: the residual stream in fp32

// A team holds one row (or group): a power of two up to 32 lanes of a warp, or all warps of the CTA.
struct Team {
  int size;
  float2* sm;  // 2 x 32; reductions take turns between two of them, so one barrier each is enough
  int turn = 0;
  template <typename Op>
  static __device__ __forceinline__ float over_warp(float v, Op op) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
  }
  // The sum of s and the maximum of m (either may be left out) over the team, of values that are not negative: 0 adds nothing.
  template <bool SUM, bool MAX>
  __device__ __forceinline__ void reduce(float& s, float& m) {
    auto add = [](float a, float b) { return a + b; };
    auto max = [](float a, float b) { return max_nan(a, b); };
    if (size < 32) {
      for (int k = size >> 1; k; k >>= 1) {
        if constexpr (SUM) s = add(s, __shfl_xor_sync(0xffffffffu, s, k));
        if constexpr (MAX) m = max(m, __shfl_xor_sync(0xffffffffu, m, k));
      }
      return;
    }
    if constexpr (SUM) s = over_warp(s, add);
    if constexpr (MAX) m = over_warp(m, max);
    if (size > 32) {
      float2* part = sm + 32 * turn;
      turn ^= 1;
      const int lane = threadIdx.x & 31;
      if (lane == 0) part[threadIdx.x >> 5] = make_float2(s, m);
      __syncthreads();
      const float2 of = lane < size >> 5 ? part[lane] : make_float2(0.f, 0.f);
      if constexpr (SUM) s = over_warp(of.x, add);
      if constexpr (MAX) m = over_warp(of.y, max);
    }
  }
};

// A thread has NV packs of VEC channels. OFF: a row may start inside a pack, the rows of all tensors at the same distance
// behind its boundary; the first and the last pack of a row then hold channels that are not the row's.
template <int VEC, bool OFF>
struct Place {
  int c, n;  // first channel, channels of the row
  __device__ __forceinline__ bool any() const { return OFF ? c > -VEC && c < n : c < n; }
  __device__ __forceinline__ bool all() const { return !OFF || (c >= 0 && c + VEC <= n); }
  __device__ __forceinline__ bool has(int i) const { return !OFF || ((unsigned)(c + i) < (unsigned)n); }
};

// A vector of parameters, dense. Rows that start inside a pack would read theirs one by one from addresses VEC floats apart,
// each load eight lines: these are put into shared memory once a CTA, a float of padding behind every 32, so that the lanes'
// floats lie in different banks (post-norm, sum and norm of 1021 x 2561: 12.2 -> 11.0 us).
template <int VEC, bool OFF>
struct Params {
  const float* p;
  static __host__ __device__ constexpr unsigned slot(unsigned c) { return c + c / 32; }
  static __host__ __device__ constexpr unsigned slots(int n) { return slot(n + 2 * VEC) + 1; }  // zeros before and behind
  __device__ __forceinline__ float* stage(float* to, int n) {
    if (p == nullptr) return to;
    for (int c = threadIdx.x - VEC; c < n + VEC; c += blockDim.x) to[slot(c + VEC)] = (unsigned)c < (unsigned)n ? __ldg(p + c) : 0.f;
    p = to;
    return to + slots(n);
  }
  __device__ __forceinline__ void get(int c0, const Place<VEC, OFF>& at, float (&x)[VEC]) const {
    if constexpr (OFF) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = p[slot(at.c + i + VEC)];
    } else if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + c0 + at.c + i));
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
      }
    } else {
      x[0] = __ldg(p + c0 + at.c);
    }
  }
};
template <typename TO, int VEC, bool OFF>
__device__ __forceinline__ void store_row(TO* row, const Place<VEC, OFF>& at, const float (&y)[VEC]) {
  if (at.all()) {
    constexpr int PV = VEC * sizeof(TO) > 16 ? 16 / sizeof(TO) : VEC;
#pragma unroll
    for (int k = 0; k < VEC; k += PV) {
      float f[PV];
#pragma unroll
      for (int i = 0; i < PV; ++i) f[i] = y[k + i];
      Pack<TO, PV> v;
      v.set(f);
      store_pack(row + at.c + k, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (at.has(i)) row[at.c + i] = from_f32<TO>(y[i]);
  }
}
template <typename T, int VEC, bool OFF>
__device__ __forceinline__ void store_as(void* base, size_t at_row, int dtype, const Place<VEC, OFF>& at, const float (&y)[VEC]) {
  if (dtype == (std::is_same_v<T, float> ? LQ_F32 : std::is_same_v<T, __half> ? LQ_F16 : LQ_BF16)) store_row(reinterpret_cast<T*>(base) + at_row, at, y);
  else if (dtype == LQ_F32) store_row(reinterpret_cast<float*>(base) + at_row, at, y);
  else if (dtype == LQ_F16) store_row(reinterpret_cast<__half*>(base) + at_row, at, y);
  else store_row(reinterpret_cast<__nv_bfloat16*>(base) + at_row, at, y);
}

// CTAs walk over the rows; a row's loads are requested while the one before is summed and stored. The register caps leave room for
// two CTAs an SM at two loads a thread (16384 x 2560, residual and norm: 56.6 us; with 112 registers and one CTA 61.5; capped
// at 64, which spills, 85), and for the widest CTA of each form.
template <typename T, int VEC, int NV, Kind KIND, bool OFF>
__global__ void __launch_bounds__(NV == 1 && !OFF || NV * VEC == 4 ? 1024 : NV == 1 ? 384 : NV == 2 ? 320 : 512, NV == 2 ? 2 : 1) norm_kernel(const lq_norm_problem p, int team_size, long long units) {
  pdl_enter();
  constexpr bool SECOND = KIND != PLAIN;
  using R = std::conditional_t<KIND == ADD32, float, T>;  // of the second input: the residual or the gate
  __shared__ float2 sm[2 * 32];
  const int rank = threadIdx.x % team_size, per_row = p.D / p.group;
  const long long step = (long long)gridDim.x * (blockDim.x / team_size);
  Team team{team_size, sm};
  const float inv_n = 1.0f / (float)p.group;
  const bool has_second = KIND == GATED || p.residual != nullptr;
  Params<VEC, OFF> weight{p.weight}, post_weight{p.post_weight}, scale_vec{p.scale_vec};
  if constexpr (OFF) {
    extern __shared__ float params[];
    float* at = params;
    for (Params<VEC, OFF>* w : {&post_weight, &scale_vec, &weight}) at = w->stage(at, p.D);
    __syncthreads();
  }

  Pack<T, VEC> raw[NV];
  constexpr int RV = VEC * sizeof(R) > 16 ? 16 / sizeof(R) : VEC;
  Pack<R, RV> raw2[SECOND ? NV : 1][SECOND ? VEC / RV : 1];
  auto place = [&](const T* x, int j) {
    const int off = OFF ? (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (VEC - 1)) : 0;
    return Place<VEC, OFF>{(j * team_size + rank) * VEC - off, p.group};
  };
  auto row_of = [&](long long unit, long long& row, int& c0) {
    row = per_row == 1 ? unit : unit / per_row;
    c0 = per_row == 1 ? 0 : (int)(unit - row * per_row) * p.group;
  };
  auto request = [&](long long unit) {
    if (unit >= units) return;
    long long row;
    int c0;
    row_of(unit, row, c0);
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride + c0;
    const R* r = nullptr;
    if constexpr (KIND == GATED) r = reinterpret_cast<const R*>(p.gate) + row * p.gate_stride + c0;
    else if constexpr (SECOND) r = reinterpret_cast<const R*>(p.residual) + row * p.residual_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Place<VEC, OFF> at = place(x, j);
      if (!at.any()) continue;
      raw[j] = load_pack<T, VEC>(x + at.c);
      if constexpr (SECOND) {
        if (has_second) {
#pragma unroll
          for (int k = 0; k < VEC / RV; ++k) raw2[j][k] = load_pack<R, RV>(r + at.c + k * RV);
        }
      }
    }
  };

  long long unit = (long long)blockIdx.x * (blockDim.x / team_size) + threadIdx.x / team_size;
  const long long rounds = (units - (long long)blockIdx.x * (blockDim.x / team_size) + step - 1) / step;  // the same for all teams: lanes without a row take part
#pragma unroll
  for (int j = 0; j < NV; ++j) {  // packs behind the last stay zero
    raw[j].zero();
    if constexpr (SECOND) {
#pragma unroll
      for (int k = 0; k < VEC / RV; ++k) raw2[j][k].zero();
    }
  }
  request(unit);
  for (long long round = 0; round < rounds; ++round, unit += step) {
    const bool live = unit < units;
    long long row;
    int c0;
    row_of(live ? unit : 0, row, c0);
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride + c0;
    float v[NV][VEC], g[SECOND ? NV : 1][VEC];
    Place<VEC, OFF> at[NV];
    bool on[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      at[j] = place(x, j);
      on[j] = live && at[j].any();
      raw[j].get(v[j]);
      if constexpr (SECOND) {
#pragma unroll
        for (int k = 0; k < VEC / RV; ++k) {
          float f[RV];
          raw2[j][k].get(f);
#pragma unroll
          for (int i = 0; i < RV; ++i) g[j][k * RV + i] = f[i];
        }
      }
      if (OFF && !at[j].all()) {  // channels of the rows next to this one
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (!at[j].has(i)) {
            v[j][i] = 0.f;
            if constexpr (SECOND) g[j][i] = 0.f;
          }
      }
    }
    request(unit + step);
    auto largest = [&]() {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) m = max_nan(m, fabsf(v[j][i]));
      return m;
    };
    // v <- v w / rms(v), `last` what multiplies it besides. The weights come before the sum is known, which leaves one product
    // behind the wait for it; the largest |v w| joins the sum's way, and times 1 / rms is the row's amax.
    float amax = 0.f;
    auto normed = [&](const Params<VEC, OFF>& w, auto with_max, auto last) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s = fmaf(v[j][i], v[j][i], s);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        float ww[VEC];
        w.get(c0, at[j], ww);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] *= ww[i];
      }
      last();
      constexpr bool MAX = decltype(with_max)::value;
      if constexpr (MAX) amax = largest();
      team.template reduce<true, MAX>(s, amax);
      const float f = rsqrtf(fmaf(s, inv_n, p.eps));
      amax *= f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] *= f;
    };
    auto out_normed = [&](auto last) {
      if (p.codes) normed(weight, std::true_type{}, last);
      else normed(weight, std::false_type{}, last);
    };

    if constexpr (KIND == ADD || KIND == ADD32) {
      if (p.post_weight) normed(post_weight, std::false_type{}, [] {});
      if (has_second) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!on[j]) continue;
          float s[VEC];
          if (p.scale_vec) scale_vec.get(c0, at[j], s);
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[j][i] = fmaf(p.scale_vec ? s[i] * p.residual_scale : p.residual_scale, v[j][i], g[j][i]);
          store_row(reinterpret_cast<R*>(p.residual_out) + (size_t)row * p.D, at[j], v[j]);
        }
      }
      if (p.weight) out_normed([] {});
    } else if constexpr (KIND == GATED) {
      auto gate = [&]() {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[j][i] *= silu(g[j][i]);
      };
      if (p.gate_first) gate();
      out_normed([&] {
        if (!p.gate_first) gate();
      });
    }
    if (p.codes) {
      if constexpr (KIND == PLAIN) {
        float none = 0.f;
        amax = largest();
        team.template reduce<false, true>(none, amax);
      }
      float inv;
      const float scale = row_scale(amax, inv);
      if (live && rank == 0) p.scale[row] = scale;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        int8_t* out = p.codes + row * p.codes_stride + at[j].c;
        if constexpr (VEC == 1 || OFF) {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (at[j].has(i)) out[i] = (int8_t)row_code(v[j][i], inv);
        } else {
          uint32_t w[VEC / 4];
#pragma unroll
          for (int i = 0; i < VEC; i += 4)
            w[i / 4] = pack_sat_s8x2(row_code(v[j][i + 1], inv), row_code(v[j][i], inv), pack_sat_s8x2(row_code(v[j][i + 3], inv), row_code(v[j][i + 2], inv), 0u));
          if constexpr (VEC == 8) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
          else *reinterpret_cast<uint32_t*>(out) = w[0];
        }
      }
    } else if (p.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on[j]) store_as<T>(p.y, (size_t)row * p.D + c0, p.out_dtype, at[j], v[j]);
    }
  }
}

// Codes of rows longer than a CTA's registers hold: a CTA a row, which is read twice, the second time out of L2: 8192 x
// 28672 bf16 123 us (5.7 TB/s of one read and the codes), 8192 x 28673, a value a load, 277 us.
template <typename T, int VEC>
__global__ void __launch_bounds__(512) quantize_long_kernel(const lq_norm_problem p) {
  pdl_enter();
  __shared__ float2 sm[2 * 32];
  Team team{512, sm};
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
    int8_t* out = p.codes + row * p.codes_stride;
    float v[VEC], none = 0.f, amax = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x * VEC; c < p.D; c += 512 * VEC) {
      load_pack<T, VEC>(x + c).get(v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) amax = max_nan(amax, fabsf(v[i]));
    }
    team.template reduce<false, true>(none, amax);
    float inv;
    const float scale = row_scale(amax, inv);
    if (threadIdx.x == 0) p.scale[row] = scale;
#pragma unroll 4
    for (int c = threadIdx.x * VEC; c < p.D; c += 512 * VEC) {
      load_pack<T, VEC>(x + c).get(v);
      Pack<int8_t, VEC> q;
#pragma unroll
      for (int i = 0; i < VEC; ++i) q.v[i] = (int8_t)row_code(v[i], inv);
      store_pack(out + c, q);
    }
  }
}
template <typename T>
static int run_long(const lq_norm_problem* p, cudaStream_t st) {
  constexpr int FULL = 16 / sizeof(T);
  Alignment a;
  const bool wide = a.at(p->x).pitch(p->x_stride, sizeof(T)).pitch(p->D, sizeof(T)).bytes() == 16;
  const int most = 4 * sm_count(), ctas = p->rows < most ? p->rows : most;
  if (wide) launch(quantize_long_kernel<T, FULL>, dim3(ctas), dim3(512), 0, st, *p);
  else launch(quantize_long_kernel<T, 1>, dim3(ctas), dim3(512), 0, st, *p);
  return check_launch("quantize_long_kernel");
}

template <typename T, Kind KIND, int VEC, int NV, bool OFF>
static int launch_as(const lq_norm_problem* p, int packs, cudaStream_t st) {
  const int need = (packs + NV - 1) / NV;
  int team = 1;
  while (team < need && team < 32) team *= 2;
  if (need > 32) team = (need + 31) / 32 * 32;
  const int threads = team > 32 ? team : 128;  // teams of several warps have the CTA's barrier and its sums to themselves
  const long long units = (long long)p->rows * (p->D / p->group), per_cta = threads / team;
  const long long ctas = (units + per_cta - 1) / per_cta;
  int per_sm = 0;
  auto kern = norm_kernel<T, VEC, NV, KIND, OFF>;
  const int params = (p->weight != nullptr) + (p->post_weight != nullptr) + (p->scale_vec != nullptr);
  // The opt-in is the most that any call needs (198 KB): it belongs to the kernel on its device, and another thread's smaller call
  // between this one's opt-in and its launch would have the launch refused.
  const int smem = OFF ? params * (int)Params<VEC, OFF>::slots(p->D) * (int)sizeof(float) : 0;
  constexpr int most_smem = 3 * (int)Params<VEC, OFF>::slots(MOST) * (int)sizeof(float);
  cudaError_t e = OFF ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem) : cudaSuccess;
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
  if (e != cudaSuccess) return fail(LQ_ERR_LAUNCH, "norm: %s", cudaGetErrorString(e));
  const long long most = (long long)sm_count() * per_sm;
  launch(kern, dim3((unsigned)(ctas < most ? ctas : most)), dim3(threads), smem, st, *p, team, units);
  return check_launch("norm_kernel");
}
// Registers hold the row, the next one on its way: two loads a thread and input where two CTAs of such threads share an SM (up to
// 640 packs), four behind that. bf16, gated norm of 32768 x 5120: 1, 2, 4 loads 289, 182, 234 us; 20480 x 8192: 246, 233 (one
// CTA an SM), 229, with INT8 outputs 286, 256, 231. 64 x 5120: 3.1, 2.8 us for one and two loads.
template <typename T, Kind KIND, int VEC, bool OFF>
static int launch_vec(const lq_norm_problem* p, cudaStream_t st) {
  const int packs = (p->group + VEC - 1) / VEC + OFF;
  if constexpr (VEC == 1) {
    if (packs <= 1024) return launch_as<T, KIND, 1, 4, OFF>(p, packs, st);
    if (packs <= MOST) return launch_as<T, KIND, 1, 32, OFF>(p, packs, st);
  } else if constexpr (OFF) {
    if (packs <= 384) return launch_as<T, KIND, VEC, 1, OFF>(p, packs, st);
    if (packs <= 640) return launch_as<T, KIND, VEC, 2, OFF>(p, packs, st);
    return launch_as<T, KIND, VEC, 32 / VEC, OFF>(p, packs, st);
  } else {
    if (packs <= 32) return launch_as<T, KIND, VEC, 1, OFF>(p, packs, st);
    if (packs <= 640) return launch_as<T, KIND, VEC, 2, OFF>(p, packs, st);
    if (packs <= 512 * 32 / VEC) return launch_as<T, KIND, VEC, 32 / VEC, OFF>(p, packs, st);
  }
  return fail(LQ_ERR_UNSUPPORTED, "norm over %d channels (at most %d)", p->group, MOST);
}
template <typename T, Kind KIND>
static int run_kind(const lq_norm_problem* p, cudaStream_t st) {
  constexpr int FULL = 16 / sizeof(T), S = sizeof(T);
  // every row of every tensor on a pack's boundary, the codes' on FULL bytes
  Alignment in, params, y;
  in.at(p->x).pitch(p->x_stride, S).pitch(p->group, S);
  if (p->gate) in.at(p->gate).pitch(p->gate_stride, S);
  params.at(p->weight).at(p->post_weight).at(p->scale_vec);
  if (KIND == ADD32) params.at(p->residual).pitch(p->residual_stride, 4).at(p->residual_out).pitch(p->D, 4);
  else if (p->residual) in.at(p->residual).pitch(p->residual_stride, S).at(p->residual_out);
  const int so = dtype_bytes(p->out_dtype), out = so * FULL;
  y.at(p->y).pitch(p->D, so).pitch(p->group, so);
  if (in.bytes() == 16 && params.bytes() == 16 && (p->y == nullptr || y.bytes() >= (out < 16 ? out : 16))) return launch_vec<T, KIND, FULL, false>(p, st);
  // rows of a length that is no multiple of a pack: the tensors' rows all at the same distance behind a boundary
  if constexpr (KIND != ADD32) {
    auto alike = [&](const void* t, long long pitch, int size) {
      return t == nullptr || (size == S && ((pitch - p->x_stride) * S & 15) == 0 && ((reinterpret_cast<uintptr_t>(t) ^ reinterpret_cast<uintptr_t>(p->x)) & 15) == 0);
    };
    if (p->group == p->D && p->D <= MOST - FULL && alike(p->gate, p->gate_stride, S) && alike(p->residual, p->residual_stride, S) &&
        alike(p->residual_out, p->D, S) && alike(p->y, p->D, so))
      return launch_vec<T, KIND, FULL, true>(p, st);
  }
  return launch_vec<T, KIND, 1, false>(p, st);
}
enum Form { NORM, GATE, CODES };
static int run(const lq_norm_problem* p, Form form, const char* what, cudaStream_t st) {
  return with_dtype(p->dtype, what, [&](auto t) {
    using T = decltype(t);
    if (form == GATE) return run_kind<T, GATED>(p, st);
    if (form == CODES) return p->D > MOST ? run_long<T>(p, st) : run_kind<T, PLAIN>(p, st);
    if constexpr (!std::is_same_v<T, float>) {
      if (p->residual && p->residual_f32) return run_kind<T, ADD32>(p, st);
    }
    return run_kind<T, ADD>(p, st);
  });
}

static int check(const lq_norm_problem* p, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->rows < 0 || p->D <= 0 || p->group <= 0 || p->D % p->group || !fits(p->D)) return fail(LQ_ERR_SHAPE, "%s: rows=%d D=%d group=%d", what, p->rows, p->D, p->group);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32 || p->out_dtype < LQ_F16 || p->out_dtype > LQ_F32)
    return fail(LQ_ERR_UNSUPPORTED, "%s: dtype %d -> %d", what, p->dtype, p->out_dtype);
  if (p->rows > 0 && !p->x) return fail(LQ_ERR_NULL, "%s: x is null", what);
  if (p->codes) {
    if (!p->scale) return fail(LQ_ERR_NULL, "%s: codes without a place for their scales", what);
    if (p->group != p->D) return fail(LQ_ERR_UNSUPPORTED, "%s: codes of rows normed in groups", what);
    if (p->codes_stride % 16 || (reinterpret_cast<uintptr_t>(p->codes) & 15u) || p->codes_stride < p->D)
      return fail(LQ_ERR_ALIGN, "%s: rows of codes start on 16-byte boundaries (pitch %lld)", what, p->codes_stride);
  }
  return LQ_OK;
}

}  // namespace norm
}  // namespace lq

extern "C" int lq_rms_norm(const lq_norm_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = norm::check(p, "rms_norm")) return e;
  if (p->group != p->D) return fail(LQ_ERR_UNSUPPORTED, "rms_norm: groups of %d channels", p->group);
  if (p->rows == 0) return LQ_OK;
  if ((p->residual == nullptr) != (p->residual_out == nullptr)) return fail(LQ_ERR_NULL, "rms_norm: a residual and the place for the sum go together");
  if ((p->y || p->codes) != (p->weight != nullptr)) return fail(LQ_ERR_NULL, "rms_norm: an output and its weight go together");
  if (!p->weight && !p->residual) return fail(LQ_ERR_NULL, "rms_norm: nothing to compute");
  if (p->post_weight && !p->residual) return fail(LQ_ERR_NULL, "rms_norm: post_weight without a residual");
  return norm::run(p, norm::NORM, "rms_norm", (cudaStream_t)stream);
}

extern "C" int lq_gated_rms_norm(const lq_norm_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = norm::check(p, "gated_rms_norm")) return e;
  if (p->rows == 0) return LQ_OK;
  if (!p->gate || !p->weight || !(p->y || p->codes)) return fail(LQ_ERR_NULL, "gated_rms_norm: gate, weight and an output must be non-null");
  if (p->residual || p->post_weight) return fail(LQ_ERR_UNSUPPORTED, "gated_rms_norm takes no residual");
  return norm::run(p, norm::GATE, "gated_rms_norm", (cudaStream_t)stream);
}

extern "C" int lq_quantize_rows(const void* x, int dtype, int rows, int D, long long x_stride, int8_t* codes, long long codes_stride, float* scale,
                                lq_stream stream) {
  using namespace lq;
  lq_norm_problem p = {};
  p.rows = rows; p.D = p.group = D;
  p.dtype = p.out_dtype = dtype;
  p.x = x; p.x_stride = x_stride; p.codes = codes; p.codes_stride = codes_stride; p.scale = scale;
  if (int e = norm::check(&p, "quantize_rows")) return e;
  if (rows == 0) return LQ_OK;
  if (!codes) return fail(LQ_ERR_NULL, "quantize_rows: codes is null");
  return norm::run(&p, norm::CODES, "quantize_rows", (cudaStream_t)stream);
}
