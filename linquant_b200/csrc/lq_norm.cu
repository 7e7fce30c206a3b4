// Norms around a block, and the row quantiser of the INT8 products.
//
//   lq_rms_norm         r = residual + alpha P(x),  P(x) = x or norm(x) post_weight;   y = norm(r) weight
//   lq_gated_rms_norm   y = norm(x silu(gate)) weight,  or  norm(x) weight silu(gate)
//   lq_quantize_rows    y = x
//   norm(v) = v / sqrt(mean(v^2) + eps) over a row (or over each group of its channels); y leaves as f16 / bf16 / f32 or as
//   INT8 codes with one scale a row (amax / 127).
//
// Memory-bound: every input is read once into registers (VEC values a load, NV loads a thread), the sums of a row are taken
// in fp32 by the team of threads that holds it, and y, r and the codes are written once.
#include "lq_layer.cuh"

namespace lq {

namespace norm {

enum Kind { ADD, GATED, PLAIN };

// A team holds one row (or group): a power of two up to 32 lanes of a warp, or all warps of the CTA.
struct Team {
  int size, rank;
  float* sm;  // 32 floats per reduction, each reduction its own
  template <typename Op>
  __device__ __forceinline__ float reduce(float v, Op op) {
    for (int m = min(size, 32) >> 1; m; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    if (size > 32) {
      const int warp = threadIdx.x >> 5, nwarps = size >> 5;
      if ((threadIdx.x & 31) == 0) sm[warp] = v;
      __syncthreads();
      v = sm[0];
      for (int w = 1; w < nwarps; ++w) v = op(v, sm[w]);
      sm += 32;
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v) { return reduce(v, [](float a, float b) { return a + b; }); }
  __device__ __forceinline__ float max(float v) { return reduce(v, [](float a, float b) { return max_nan(a, b); }); }
};

template <int VEC>
__device__ __forceinline__ void load_f32(const float* p, int c, float (&x)[VEC]) {  // parameters: dense, 16-byte aligned where VEC > 1
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + c + i));
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = __ldg(p + c + i);
  }
}
template <int VEC>
__device__ __forceinline__ void store_as(void* base, size_t at, int dtype, const float (&y)[VEC]) {
  if (dtype == LQ_F32) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4)
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) reinterpret_cast<float*>(base)[at + i] = y[i];
    }
  } else if (dtype == LQ_F16) {
    Pack<__half, VEC> v;
    v.set(y);
    store_pack(reinterpret_cast<__half*>(base) + at, v);
  } else {
    Pack<__nv_bfloat16, VEC> v;
    v.set(y);
    store_pack(reinterpret_cast<__nv_bfloat16*>(base) + at, v);
  }
}

template <typename T, int VEC, int NV, Kind KIND>
__global__ void __launch_bounds__(NV * VEC > 16 ? 512 : 1024) norm_kernel(const lq_norm_problem p, int team_size, long long units) {
  pdl_enter();
  __shared__ float sm[3 * 32];
  const int rank = threadIdx.x % team_size;
  const long long unit = (long long)blockIdx.x * (blockDim.x / team_size) + threadIdx.x / team_size;
  const bool live = unit < units;  // lanes of a team that has no row still take part in the shuffles
  const int per_row = p.D / p.group;
  const long long row = live ? unit / per_row : 0;
  const int c0 = (int)(live ? unit - row * per_row : 0) * p.group;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride + c0;
  Team team{team_size, rank, sm};
  const float inv_n = 1.0f / (float)p.group;

  float v[NV][VEC], g[KIND == GATED ? NV : 1][VEC];
  bool on[NV];
  {
    Pack<T, VEC> raw[NV], rawg[KIND == GATED ? NV : 1];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team_size + rank) * VEC;
      on[j] = live && c < p.group;
      raw[j].zero();
      if (on[j]) raw[j] = load_pack<T, VEC>(x + c);
      if constexpr (KIND == GATED) {
        rawg[j].zero();
        if (on[j]) rawg[j] = load_pack<T, VEC>(reinterpret_cast<const T*>(p.gate) + row * p.gate_stride + c0 + c);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      raw[j].get(v[j]);
      if constexpr (KIND == GATED) rawg[j].get(g[j]);
    }
  }
  auto rms = [&]() {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s = fmaf(v[j][i], v[j][i], s);
    return rsqrtf(fmaf(team.sum(s), inv_n, p.eps));
  };
  auto times = [&](float f, const float* w) {  // v f w
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!on[j]) continue;
      float ww[VEC];
      load_f32<VEC>(w, c0 + (j * team_size + rank) * VEC, ww);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = v[j][i] * f * ww[i];
    }
  };

  if constexpr (KIND == ADD) {
    if (p.post_weight) times(rms(), p.post_weight);
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        const int c = (j * team_size + rank) * VEC;
        float r[VEC], s[VEC];
        if (p.residual_f32) load_f32<VEC>(reinterpret_cast<const float*>(p.residual) + row * p.residual_stride, c, r);
        else load_pack<T, VEC>(reinterpret_cast<const T*>(p.residual) + row * p.residual_stride + c).get(r);
        if (p.scale_vec) load_f32<VEC>(p.scale_vec, c, s);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = fmaf(p.scale_vec ? s[i] * p.residual_scale : p.residual_scale, v[j][i], r[i]);
        if (p.residual_f32) store_as<VEC>(p.residual_out, (size_t)row * p.D + c, LQ_F32, v[j]);
        else store_as<VEC>(p.residual_out, (size_t)row * p.D + c, std::is_same_v<T, float> ? LQ_F32 : std::is_same_v<T, __half> ? LQ_F16 : LQ_BF16, v[j]);
      }
    }
    if (p.weight) times(rms(), p.weight);
  } else if constexpr (KIND == GATED) {
    auto gate = [&]() {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] *= silu(g[j][i]);
    };
    if (p.gate_first) gate();
    times(rms(), p.weight);
    if (!p.gate_first) gate();
  }
  if (p.codes) {
    float amax = 0.f, inv;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (on[j])
#pragma unroll
        for (int i = 0; i < VEC; ++i) amax = max_nan(amax, fabsf(v[j][i]));
    const float scale = row_scale(team.max(amax), inv);
    if (live && rank == 0) p.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!on[j]) continue;
      int8_t* out = p.codes + row * p.codes_stride + (j * team_size + rank) * VEC;
      if constexpr (VEC == 1) {
        out[0] = (int8_t)q8(v[j][0], inv, 127.f);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
          reinterpret_cast<uint32_t*>(out)[i / 4] = q8x4_127(v[j][i], v[j][i + 1], v[j][i + 2], v[j][i + 3], inv);
      }
    }
  } else if (p.y) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (on[j]) store_as<VEC>(p.y, (size_t)row * p.D + c0 + (j * team_size + rank) * VEC, p.out_dtype, v[j]);
  }
}

// Registers hold the row: the fewest loads a thread that leave a team of at most 256 threads (a row is then in flight from
// many small CTAs), more where the row is longer.
template <typename T, Kind KIND, int VEC, int NV>
static int launch_as(const lq_norm_problem* p, int packs, cudaStream_t st) {
  const int need = (packs + NV - 1) / NV;
  int team = 1;
  while (team < need && team < 32) team *= 2;
  if (need > 32) team = (need + 31) / 32 * 32;
  const int threads = team > 32 ? team : 128;  // teams of several warps have the CTA's barrier and its sums to themselves
  const long long units = (long long)p->rows * (p->D / p->group), per_cta = threads / team;
  const long long ctas = (units + per_cta - 1) / per_cta;
  if (ctas >= (1ll << 31)) return fail(LQ_ERR_SHAPE, "norm: rows=%d D=%d group=%d", p->rows, p->D, p->group);
  launch(norm_kernel<T, VEC, NV, KIND>, dim3((unsigned)ctas), dim3(threads), 0, st, *p, team, units);
  return check_launch("norm_kernel");
}
template <typename T, Kind KIND, int VEC>
static int launch_vec(const lq_norm_problem* p, cudaStream_t st) {
  const int packs = (p->group + VEC - 1) / VEC;
  constexpr int MOST = VEC == 1 ? 32 : 32 / VEC;  // 32 values a thread
  if (packs <= 256) return launch_as<T, KIND, VEC, 1>(p, packs, st);
  if (packs <= 1024) return launch_as<T, KIND, VEC, MOST < 4 ? MOST : 4>(p, packs, st);
  if (packs <= 512 * MOST) return launch_as<T, KIND, VEC, MOST>(p, packs, st);
  return fail(LQ_ERR_UNSUPPORTED, "norm over %d channels (at most %d)", p->group, 16384);
}
template <Kind KIND>
static int run(const lq_norm_problem* p, const char* what, cudaStream_t st) {
  return with_dtype(p->dtype, what, [&](auto t) {
    using T = decltype(t);
    constexpr int FULL = 16 / sizeof(T), S = sizeof(T);
    const int out = dtype_bytes(p->out_dtype) * FULL, res = p->residual_f32 ? 4 : S;
    Alignment in, params;
    in.at(p->x).pitch(p->x_stride, S).pitch(p->group, S);
    if (p->gate) in.at(p->gate).pitch(p->gate_stride, S);
    params.at(p->weight).at(p->post_weight).at(p->scale_vec);
    if (p->residual_f32) params.at(p->residual).pitch(p->residual_stride, 4).at(p->residual_out).pitch(p->D, 4);
    else if (p->residual) in.at(p->residual).pitch(p->residual_stride, res).at(p->residual_out);
    Alignment y;
    y.at(p->y).pitch(p->D, dtype_bytes(p->out_dtype)).pitch(p->group, dtype_bytes(p->out_dtype));
    Alignment codes;
    codes.at(p->codes).pitch(p->codes_stride, 1);
    const bool wide = in.bytes() == 16 && params.bytes() == 16 && (p->y == nullptr || y.bytes() >= (out < 16 ? out : 16)) && codes.bytes() == 16;
    return wide ? launch_vec<T, KIND, FULL>(p, st) : launch_vec<T, KIND, 1>(p, st);
  });
}

static int check(const lq_norm_problem* p, const char* what) {
  if (!p) return fail(LQ_ERR_NULL, "%s: problem descriptor is null", what);
  if (p->rows < 0 || p->D <= 0 || p->group <= 0 || p->D % p->group) return fail(LQ_ERR_SHAPE, "%s: rows=%d D=%d group=%d", what, p->rows, p->D, p->group);
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
  return norm::run<norm::ADD>(p, "rms_norm", (cudaStream_t)stream);
}

extern "C" int lq_gated_rms_norm(const lq_norm_problem* p, lq_stream stream) {
  using namespace lq;
  if (int e = norm::check(p, "gated_rms_norm")) return e;
  if (p->rows == 0) return LQ_OK;
  if (!p->gate || !p->weight || !(p->y || p->codes)) return fail(LQ_ERR_NULL, "gated_rms_norm: gate, weight and an output must be non-null");
  if (p->residual || p->post_weight) return fail(LQ_ERR_UNSUPPORTED, "gated_rms_norm takes no residual");
  return norm::run<norm::GATED>(p, "gated_rms_norm", (cudaStream_t)stream);
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
  return norm::run<norm::PLAIN>(&p, "quantize_rows", (cudaStream_t)stream);
}
