// Group norm with an activation, channels last.
//
//   y = act((x - mean) / sqrt(var + eps) weight + bias) [silu(gate)]         mean and var over a group's values
//
// Of single tokens a group is its C = D / groups channels: a team of 8, 32 or 256 threads holds them in registers (up to four packs a
// thread, what lies behind is read again from cache), sums them, then the squares of their distances from the mean: no
// cancellation, one pass over memory.
// Over the tokens of a sequence it is T x C values, in two kernels. The first leaves for each tile of tokens and each group its mean
// and sum of squared distances (a channel's values by eights around their own mean, merged by the exact formula for two
// sets, then channels, tokens and tiles the same way); the second merges the tiles of its sequence and writes y, reading x from
// L2 where it fits there. All sums are fp32, in a fixed order.
#include "lq_layer.cuh"

namespace lq {

namespace group_norm {

constexpr int THREADS = 256, HOLD = 4;

__device__ __forceinline__ float inv_std(float var, float eps) { return 1.0f / sqrtf(var + eps); }

template <int VEC>
__device__ __forceinline__ void load_parameters(const float* p, float none, float (&x)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = none;
  } else if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = __ldg(p + i);
  }
}

template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* part) {
#pragma unroll
  for (int m = (TEAM < 32 ? TEAM : 32) / 2; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  if constexpr (TEAM > 32) {
    __syncthreads();  // the sums before have been read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TEAM / 32; ++w) v += part[w];
  }
  return v;
}

// Single tokens: one group a team, packs of VEC values
template <typename T, int VEC, int TEAM>
__global__ void __launch_bounds__(THREADS) group_norm_rows_kernel(const lq_group_norm_problem p) {
  __shared__ float part[THREADS / 32];
  constexpr int TEAMS = THREADS / TEAM;
  const int C = p.D / p.groups, packs = C / VEC, me = threadIdx.x % TEAM;
  const long long count = (long long)p.B * p.groups;
  pdl_enter();
  const long long item = (long long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
  const bool on = item < count;  // teams of a warp stay together in its shuffles
  const int row = on ? (int)(item / p.groups) : 0, c0 = on ? (int)(item - (long long)row * p.groups) * C : 0;
  const T* x = reinterpret_cast<const T*>(p.x) + (long long)row * p.x_stride_b + c0;
  const T* gate = p.gate ? reinterpret_cast<const T*>(p.gate) + (long long)row * p.gate_stride_b + c0 : nullptr;
  T* y = reinterpret_cast<T*>(p.y) + (long long)row * p.D + c0;
  const int mine = on ? packs : 0;
  Pack<T, VEC> raw[HOLD], g[HOLD];
#pragma unroll
  for (int h = 0; h < HOLD; ++h) {
    const int at = me + h * TEAM;
    raw[h].zero();
    g[h].zero();
    if (at < mine) {
      raw[h] = load_pack<T, VEC>(x + at * VEC);
      if (gate) g[h] = load_pack<T, VEC>(gate + at * VEC);
    }
  }
  float sum = 0.f;
  auto add = [&](const Pack<T, VEC>& r) {
    float v[VEC];
    r.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += v[i];
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h) add(raw[h]);
  for (int at = me + HOLD * TEAM; at < mine; at += TEAM) add(load_pack<T, VEC>(x + at * VEC));
  const float mean = team_sum<TEAM>(sum, part) / (float)C;
  sum = 0.f;
  auto square = [&](const Pack<T, VEC>& r) {
    float v[VEC];
    r.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum = fmaf(v[i] - mean, v[i] - mean, sum);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (me + h * TEAM < mine) square(raw[h]);
  for (int at = me + HOLD * TEAM; at < mine; at += TEAM) square(load_pack<T, VEC>(x + at * VEC));
  const float r = inv_std(team_sum<TEAM>(sum, part) / (float)C, p.eps);
  auto store = [&](int at, const Pack<T, VEC>& in, const Pack<T, VEC>& gin) {
    float v[VEC], w[VEC], b[VEC];
    in.get(v);
    load_parameters<VEC>(p.weight ? p.weight + c0 + at * VEC : nullptr, 1.f, w);
    load_parameters<VEC>(p.bias ? p.bias + c0 + at * VEC : nullptr, 0.f, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[i] = fmaf((v[i] - mean) * r, w[i], b[i]);
      if (p.silu) v[i] = silu(v[i]);
    }
    if (gate) {
      float z[VEC];
      gin.get(z);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= silu(z[i]);
    }
    Pack<T, VEC> out;
    out.set(v);
    store_pack(y + at * VEC, out);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (me + h * TEAM < mine) store(me + h * TEAM, raw[h], g[h]);
  for (int at = me + HOLD * TEAM; at < mine; at += TEAM) {
    Pack<T, VEC> gin;
    gin.zero();
    if (gate) gin = load_pack<T, VEC>(gate + at * VEC);
    store(at, load_pack<T, VEC>(x + at * VEC), gin);
  }
}

// ---- over the tokens of a sequence
constexpr int CHANNELS = 2048, U = 8;  // channels of a CTA at most (or one group's part), tokens in flight a thread

struct Tiles {
  int count, tokens;       // of a sequence
  int block, blocks;       // groups of a CTA; CTAs next to one another
  float2* sums;            // [B][count][groups]: mean, sum of squared distances
};

// A set of n values joins another one: the mean and sum of squared distances of both
__device__ __forceinline__ void join(float& mean, float& m2, float other_mean, float other_m2, float share, float weight) {
  const float d = other_mean - mean;  // share = n_other / n_both, weight = n n_other / n_both
  mean = fmaf(d, share, mean);
  m2 += fmaf(d * d, weight, other_m2);
}

// channels c0 .. c0 + chans of the CTA: a thread has packs of VEC channels, and of its tile the tokens r, r + rows, ..
template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) group_norm_sums_kernel(const lq_group_norm_problem p, const Tiles t) {
  __shared__ float s_mean[CHANNELS], s_m2[CHANNELS];
  const int C = p.D / p.groups, b = blockIdx.z, tile = blockIdx.x, g0 = blockIdx.y * t.block, groups = min(t.block, p.groups - g0);
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = (int)min((long long)tile * t.tokens, (long long)n), tokens = (int)min((long long)t.tokens, (long long)n - first);
  const int width = groups * C;  // one group may be wider than a CTA: its parts one after the other
  float all_mean = 0.f, all_m2 = 0.f, all_n = 0.f;
  for (int part = 0; part < width; part += CHANNELS) {
    const int chans = min(CHANNELS, width - part), packs = (chans + VEC - 1) / VEC, rows = packs < THREADS ? THREADS / packs : 1;
    const T* x = reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + first * p.x_stride_t + (long long)g0 * C + part;
    if (part > 0) __syncthreads();
    for (int i = threadIdx.x; i < packs * rows; i += THREADS) {
      const int pack = i % packs, r = i / packs;
      float mean[VEC], m2[VEC];
      int have = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) mean[v] = m2[v] = 0.f;
      for (int t0 = r; t0 < tokens; t0 += rows * U) {
        Pack<T, VEC> raw[U];
        const int more = min(U, (tokens - t0 + rows - 1) / rows);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < more) raw[u] = load_pack<T, VEC>(x + (long long)(t0 + u * rows) * p.x_stride_t + pack * VEC);
          else raw[u].zero();
        float sum[VEC], sq[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] = sq[v] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[VEC];
          raw[u].get(f);
#pragma unroll
          for (int v = 0; v < VEC; ++v) sum[v] += f[v];
        }
        const float inv = 1.f / (float)more, share = (float)more / (float)(have + more), weight = (float)have * share;
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] *= inv;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[VEC];
          raw[u].get(f);
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            if (u < more) sq[v] = fmaf(f[v] - sum[v], f[v] - sum[v], sq[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) join(mean[v], m2[v], sum[v], sq[v], share, weight);
        have += more;
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (pack * VEC + v < chans) s_mean[r * chans + pack * VEC + v] = mean[v], s_m2[r * chans + pack * VEC + v] = m2[v];
    }
    __syncthreads();
    // a warp a group: channels and token rows, each of the values it has
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, span = min(C, chans);
    for (int g = warp; g < chans / span; g += THREADS / 32) {
      const float values = (float)tokens * (float)span;
      float mean = 0.f, m2 = 0.f;
      for (int i = lane; i < rows * span; i += 32) {
        const int r = i / span;
        mean = fmaf((float)((tokens - r + rows - 1) / rows) / values, s_mean[r * chans + g * span + i % span], mean);
      }
#pragma unroll
      for (int m = 16; m; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
      for (int i = lane; i < rows * span; i += 32) {
        const int r = i / span, at = r * chans + g * span + i % span, have = (tokens - r + rows - 1) / rows;
        const float d = s_mean[at] - mean;
        if (have > 0) m2 += fmaf(d * d, (float)have, s_m2[at]);
      }
#pragma unroll
      for (int m = 16; m; m >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, m);
      if (tokens <= 0) mean = m2 = 0.f;
      if (width > CHANNELS) {  // one group: its parts meet in warp 0
        const float both = all_n + values;
        if (both > 0.f) join(all_mean, all_m2, mean, m2, values / both, all_n * (values / both));
        all_n = both;
        mean = all_mean, m2 = all_m2;
      }
      if (lane == 0 && part + CHANNELS >= width) t.sums[((size_t)b * t.count + tile) * p.groups + g0 + g] = make_float2(mean, m2);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) group_norm_apply_kernel(const lq_group_norm_problem p, const Tiles t) {
  __shared__ float s_mean[CHANNELS], s_inv[CHANNELS];  // of the CTA's groups
  const int C = p.D / p.groups, b = blockIdx.z, g0 = blockIdx.y * t.block, groups = min(t.block, p.groups - g0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = (int)min((long long)blockIdx.x * t.tokens, (long long)p.T), stop = (int)min((long long)first + t.tokens, (long long)p.T);
  for (int g = warp; g < groups; g += THREADS / 32) {
    const float2* sums = t.sums + (size_t)b * t.count * p.groups + g0 + g;
    float mean = 0.f, m2 = 0.f;
    for (int i = lane; i < t.count; i += 32) {
      const float have = (float)max(min((long long)t.tokens, (long long)n - (long long)i * t.tokens), 0ll);
      if (have > 0.f) mean = fmaf(have / (float)n, sums[(size_t)i * p.groups].x, mean);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
    for (int i = lane; i < t.count; i += 32) {
      const float have = (float)max(min((long long)t.tokens, (long long)n - (long long)i * t.tokens), 0ll);
      const float2 s = sums[(size_t)i * p.groups];
      if (have > 0.f) m2 += fmaf((s.x - mean) * (s.x - mean), have * (float)C, s.y);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, m);
    if (lane == 0) s_mean[g] = mean, s_inv[g] = inv_std(m2 / ((float)n * (float)C), p.eps);
  }
  __syncthreads();
  const int width = groups * C, packs = (width + VEC - 1) / VEC, rows = packs < THREADS ? THREADS / packs : 1;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + (long long)g0 * C;
  const T* gate = p.gate ? reinterpret_cast<const T*>(p.gate) + b * p.gate_stride_b + (long long)g0 * C : nullptr;
  T* y = reinterpret_cast<T*>(p.y) + (long long)b * p.T * p.D + (long long)g0 * C;
  for (int i = threadIdx.x; i < packs * rows; i += THREADS) {
    const int pack = i % packs, r = i / packs;
    float mean[VEC], a[VEC], c[VEC];
    load_parameters<VEC>(p.weight ? p.weight + g0 * C + pack * VEC : nullptr, 1.f, a);
    load_parameters<VEC>(p.bias ? p.bias + g0 * C + pack * VEC : nullptr, 0.f, c);
    const int g = pack * VEC / C;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const int at = C % VEC == 0 ? g : (pack * VEC + v) / C;
      mean[v] = s_mean[at];
      a[v] *= s_inv[at];
    }
    for (int t0 = first + r; t0 < stop; t0 += rows * U) {
      Pack<T, VEC> raw[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = t0 + u * rows;
        raw[u].zero();
        if (at < min(stop, n)) raw[u] = load_pack<T, VEC>(x + (long long)at * p.x_stride_t + pack * VEC);
        if (gate && at < min(stop, n)) z[u] = load_pack<T, VEC>(gate + (long long)at * p.gate_stride_t + pack * VEC);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = t0 + u * rows;
        if (at >= stop) break;
        float f[VEC];
        raw[u].get(f);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          f[v] = fmaf(f[v] - mean[v], a[v], c[v]);
          if (p.silu) f[v] = silu(f[v]);
        }
        if (gate) {
          float zf[VEC];
          z[u].get(zf);
#pragma unroll
          for (int v = 0; v < VEC; ++v) f[v] *= silu(zf[v]);
        }
        Pack<T, VEC> out;
        out.set(f);
        if (at >= n) out.zero();  // behind the sequence
        store_pack(y + (long long)at * p.D + pack * VEC, out);
      }
    }
  }
}

static int check(const lq_group_norm_problem* p) {
  if (!p) return fail(LQ_ERR_NULL, "group_norm: problem descriptor is null");
  if (p->B < 0 || p->T < 0 || p->D <= 0 || p->groups <= 0 || p->D % p->groups || !fits(p->B) || !fits(p->T) || !fits(p->D))
    return fail(LQ_ERR_SHAPE, "group_norm: B=%d T=%d D=%d groups=%d", p->B, p->T, p->D, p->groups);
  if (p->dtype < LQ_F16 || p->dtype > LQ_F32) return fail(LQ_ERR_UNSUPPORTED, "group_norm: dtype %d", p->dtype);
  if (!p->over_tokens && p->T != 1) return fail(LQ_ERR_SHAPE, "group_norm: T=%d without over_tokens", p->T);
  if (!p->over_tokens && p->lengths) return fail(LQ_ERR_SHAPE, "group_norm: lengths go with over_tokens");
  if (p->over_tokens && p->B > 65535) return fail(LQ_ERR_SHAPE, "group_norm: B=%d sequences", p->B);
  return LQ_OK;
}
// Tiles of tokens: three CTAs an SM, at least 16 tokens each
static Tiles tiles_of(const lq_group_norm_problem* p) {
  Tiles t = {};
  const int C = p->D / p->groups;
  t.block = C >= CHANNELS ? 1 : CHANNELS / C;
  if (t.block > p->groups) t.block = p->groups;
  t.blocks = (p->groups + t.block - 1) / t.block;
  const long long columns = (long long)p->B * t.blocks, room = 3ll * sm_count();
  long long count = columns > 0 ? (room + columns - 1) / columns : 1;
  const long long most = ((long long)p->T + 15) / 16;
  count = count > most ? most : count;
  count = count < 1 ? 1 : count;
  t.tokens = (int)(((long long)p->T + count - 1) / count);
  if (t.tokens < 1) t.tokens = 1;
  t.count = (int)(((long long)p->T + t.tokens - 1) / t.tokens);
  if (t.count < 1) t.count = 1;
  return t;
}

}  // namespace group_norm

}  // namespace lq

extern "C" size_t lq_group_norm_workspace_bytes(const lq_group_norm_problem* p) {
  using namespace lq::group_norm;
  if (check(p) != LQ_OK || !p->over_tokens) return 0;
  return (size_t)p->B * tiles_of(p).count * p->groups * sizeof(float2);
}

extern "C" int lq_group_norm(const lq_group_norm_problem* p, void* ws, size_t bytes, lq_stream stream) {
  using namespace lq;
  using namespace lq::group_norm;
  if (int e = group_norm::check(p)) return e;
  if (p->B == 0 || p->T == 0) return LQ_OK;
  if (!p->x || !p->y) return fail(LQ_ERR_NULL, "group_norm: x and y must be non-null");
  cudaStream_t st = (cudaStream_t)stream;
  const int C = p->D / p->groups, size = dtype_bytes(p->dtype);
  Tiles t = {};
  if (p->over_tokens) {
    t = tiles_of(p);
    if (t.blocks > 65535) return fail(LQ_ERR_SHAPE, "group_norm: D=%d groups=%d", p->D, p->groups);
    const size_t need = lq_group_norm_workspace_bytes(p);
    if (!ws || bytes < need) return fail(LQ_ERR_WORKSPACE, "group_norm: workspace of %zu bytes, %zu needed", bytes, need);
    if (reinterpret_cast<uintptr_t>(ws) & 7u) return fail(LQ_ERR_ALIGN, "group_norm: workspace must start on an 8-byte boundary");
    t.sums = reinterpret_cast<float2*>(ws);
  }
  // a pack may not leave its row (single tokens: its group), and starts on a boundary of its size in every tensor
  Alignment a;
  a.at(p->x).at(p->y).pitch(p->x_stride_b, size).pitch(p->D, size);
  if (p->gate) a.at(p->gate).pitch(p->gate_stride_b, size);
  if (p->over_tokens) {
    a.pitch(p->x_stride_t, size).pitch((long long)t.block * C, size);
    if (p->gate) a.pitch(p->gate_stride_t, size);
  } else {
    a.pitch(C, size);
  }
  const bool parameters = ((reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(p->bias)) & 15u) == 0;
  const int access = a.bytes() == 16 && parameters ? 16 : a.bytes() >= 4 ? 4 : 2;
  return with_dtype(p->dtype, "group_norm", [&](auto type) {
    using T = decltype(type);
    constexpr int FULL = 16 / sizeof(T), WORD = 4 / sizeof(T);
    auto done = [&](cudaError_t e) { return e != cudaSuccess ? fail(LQ_ERR_LAUNCH, "group_norm: %s", cudaGetErrorString(e)) : check_launch("group_norm_kernel"); };
    auto with_vec = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      if (p->over_tokens) {
        const dim3 grid(t.count, t.blocks, p->B);
        cudaError_t e = launch(group_norm_sums_kernel<T, VEC>, grid, dim3(THREADS), 0, st, *p, t);
        if (e == cudaSuccess) e = launch(group_norm_apply_kernel<T, VEC>, grid, dim3(THREADS), 0, st, *p, t);
        return done(e);
      }
      // the narrowest team that holds a group in registers
      const long long items = (long long)p->B * p->groups;
      const int packs = C / VEC, team = packs <= 8 * HOLD ? 8 : packs <= 32 * HOLD ? 32 : 256;
      const long long ctas = (items + THREADS / team - 1) / (THREADS / team);
      if (ctas > 0x7fffffffll) return fail(LQ_ERR_SHAPE, "group_norm: %lld groups", items);
      const dim3 grid((unsigned)ctas), block(THREADS);
      return done(team == 8    ? launch(group_norm_rows_kernel<T, VEC, 8>, grid, block, 0, st, *p)
                  : team == 32 ? launch(group_norm_rows_kernel<T, VEC, 32>, grid, block, 0, st, *p)
                               : launch(group_norm_rows_kernel<T, VEC, 256>, grid, block, 0, st, *p));
    };
    if (access == 16) return with_vec(std::integral_constant<int, FULL>());
    if constexpr (WORD > 1)
      if (access == 4) return with_vec(std::integral_constant<int, WORD>());
    return with_vec(std::integral_constant<int, 1>());
  });
}
