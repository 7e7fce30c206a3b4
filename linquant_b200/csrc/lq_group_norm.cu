// Group norm with an activation, channels last.
//
//   y = act((x - mean) / sqrt(var + eps) weight + bias) [silu(gate)]         mean and var over a group's values
//
// Of single tokens a group is its C = D / groups channels, held in registers by a team of threads, summed, then the squares of their
// distances from the mean: no cancellation, one pass over memory. Up to 128 packs of 16 bytes a team is 8 to 32 lanes, a thread keeps
// its channels' weights and walks over rows, several of them on their way; wider groups take a CTA (four packs a thread, what lies
// behind is read again from cache).
// Over the tokens of a sequence it is T x C values, in two kernels. The first leaves for each tile of tokens and each group its mean
// and sum of squared distances (a channel's values by eights around their own mean, merged by the exact formula for two
// sets, then channels, tokens and tiles the same way); the second merges the tiles of its sequence and writes y, reading x from
// L2 where it fits there. All sums are fp32, in a fixed order.
// 32768 x 2048 fp16 in 16 groups with a gate: 86 us, 4.7 TB/s (half of HBM's cycles, 56 % of the issue slots); without a gate, bf16: 62 to 68 us, 4.0 to 4.3 TB/s. No
// unit is full: a team requests its next rows behind the two sums of these. Over 6 x 1499 tokens x 1026 channels, ragged: 23 us, the latency of two kernels whose
// accesses are 4 bytes wide, as rows of 2052 bytes allow; a round of CTAs is best (tiles of half the tokens, two rounds: 27).
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

__device__ __forceinline__ float cta_sum(float v, float* part) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();  // the sums before have been read
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += part[w];
  return v;
}

// Single tokens, a group a team of TEAM lanes with PP packs of VEC values each; U rows on their way. The CTA has `block` groups of
// `together` rows at a time.
template <typename T, int VEC, int TEAM, int PP>
__global__ void __launch_bounds__(THREADS) group_norm_rows_kernel(const lq_group_norm_problem p, int block, int together) {
  constexpr int U = 4 / PP;
  const int C = p.D / p.groups, packs = C / VEC, team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
  const int g = blockIdx.y * block + team % block, r = team / block;
  const bool on = r < together && g < p.groups;
  const int c0 = on ? g * C : 0;
  float w[PP][VEC], b[PP][VEC];
  pdl_enter();
#pragma unroll
  for (int h = 0; h < PP; ++h) {
    const int at = me + h * TEAM;
    const bool in = on && at < packs;
    load_parameters<VEC>(in && p.weight ? p.weight + c0 + at * VEC : nullptr, 1.f, w[h]);
    load_parameters<VEC>(in && p.bias ? p.bias + c0 + at * VEC : nullptr, 0.f, b[h]);
  }
  const float inv_c = 1.f / (float)C;
  const T* x = reinterpret_cast<const T*>(p.x) + c0;
  const T* gate = p.gate ? reinterpret_cast<const T*>(p.gate) + c0 : nullptr;
  T* y = reinterpret_cast<T*>(p.y) + c0;
  for (long long row0 = (long long)blockIdx.x * together + r; row0 - r < p.B; row0 += (long long)gridDim.x * together * U) {
    Pack<T, VEC> raw[U][PP], z[U][PP];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = row0 + (long long)u * gridDim.x * together;
#pragma unroll
      for (int h = 0; h < PP; ++h) {
        const int at = me + h * TEAM;
        raw[u][h].zero();
        z[u][h].zero();
        if (on && row < p.B && at < packs) {
          raw[u][h] = load_pack<T, VEC>(x + row * p.x_stride_b + at * VEC);
          if (gate) z[u][h] = load_pack<T, VEC>(gate + row * p.gate_stride_b + at * VEC);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = row0 + (long long)u * gridDim.x * together;
      float v[PP][VEC], sum = 0.f;
#pragma unroll
      for (int h = 0; h < PP; ++h) {
        raw[u][h].get(v[h]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += v[h][i];
      }
#pragma unroll
      for (int m = TEAM / 2; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      const float mean = sum * inv_c;
      sum = 0.f;
#pragma unroll
      for (int h = 0; h < PP; ++h)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[h][i] -= mean;
          sum = me + h * TEAM < packs ? fmaf(v[h][i], v[h][i], sum) : sum;
        }
#pragma unroll
      for (int m = TEAM / 2; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      const float scale = inv_std(sum * inv_c, p.eps);
#pragma unroll
      for (int h = 0; h < PP; ++h) {
        const int at = me + h * TEAM;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[h][i] = fmaf(v[h][i] * scale, w[h][i], b[h][i]);
        if (p.silu)
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[h][i] = silu(v[h][i]);
        if (gate) {
          float f[VEC];
          z[u][h].get(f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[h][i] *= silu(f[i]);
        }
        Pack<T, VEC> out;
        out.set(v[h]);
        if (on && row < p.B && at < packs) store_pack(y + row * p.D + at * VEC, out);
      }
    }
  }
}

// Single tokens, a group a CTA: packs of VEC values
template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) group_norm_wide_kernel(const lq_group_norm_problem p) {
  constexpr int TEAM = THREADS;
  __shared__ float part[THREADS / 32];
  const int C = p.D / p.groups, packs = C / VEC, me = threadIdx.x;
  pdl_enter();
  const int row = blockIdx.x / p.groups, c0 = (blockIdx.x - row * p.groups) * C;
  const T* x = reinterpret_cast<const T*>(p.x) + (long long)row * p.x_stride_b + c0;
  const T* gate = p.gate ? reinterpret_cast<const T*>(p.gate) + (long long)row * p.gate_stride_b + c0 : nullptr;
  T* y = reinterpret_cast<T*>(p.y) + (long long)row * p.D + c0;
  Pack<T, VEC> raw[HOLD], g[HOLD];
#pragma unroll
  for (int h = 0; h < HOLD; ++h) {
    const int at = me + h * TEAM;
    raw[h].zero();
    g[h].zero();
    if (at < packs) {
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
  for (int at = me + HOLD * TEAM; at < packs; at += TEAM) add(load_pack<T, VEC>(x + at * VEC));
  const float mean = cta_sum(sum, part) / (float)C;
  sum = 0.f;
  auto square = [&](const Pack<T, VEC>& r) {
    float v[VEC];
    r.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum = fmaf(v[i] - mean, v[i] - mean, sum);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (me + h * TEAM < packs) square(raw[h]);
  for (int at = me + HOLD * TEAM; at < packs; at += TEAM) square(load_pack<T, VEC>(x + at * VEC));
  const float r = inv_std(cta_sum(sum, part) / (float)C, p.eps);
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
    if (me + h * TEAM < packs) store(me + h * TEAM, raw[h], g[h]);
  for (int at = me + HOLD * TEAM; at < packs; at += TEAM) {
    Pack<T, VEC> gin;
    gin.zero();
    if (gate) gin = load_pack<T, VEC>(gate + at * VEC);
    store(at, load_pack<T, VEC>(x + at * VEC), gin);
  }
}

// ---- over the tokens of a sequence
constexpr int CHANNELS = 2048, WIDE = 640;  // channels of a CTA at most (or one group's part); threads at most
template <int VEC>
constexpr int kInFlight = VEC >= 4 ? 4 : 8;  // tokens on their way, a thread

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
__global__ void __launch_bounds__(WIDE, VEC >= 4 ? 1 : 2) group_norm_sums_kernel(const lq_group_norm_problem p, const Tiles t) {
  constexpr int U = kInFlight<VEC>;
  constexpr int ENTRIES = WIDE * VEC > CHANNELS ? WIDE * VEC : CHANNELS;  // a channel and token row each
  __shared__ float s_mean[ENTRIES], s_m2[ENTRIES];
  const int C = p.D / p.groups, b = blockIdx.z, tile = blockIdx.x, g0 = blockIdx.y * t.block, groups = min(t.block, p.groups - g0);
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = (int)min((long long)tile * t.tokens, (long long)n), tokens = (int)min((long long)t.tokens, (long long)n - first);
  const int width = groups * C;  // one group may be wider than a CTA: its parts one after the other
  float all_mean = 0.f, all_m2 = 0.f, all_n = 0.f;
  for (int part = 0; part < width; part += CHANNELS) {
    const int chans = min(CHANNELS, width - part), packs = (chans + VEC - 1) / VEC, rows = max((int)blockDim.x / packs, 1);
    const T* x = reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + first * p.x_stride_t + (long long)g0 * C + part;
    if (part > 0) __syncthreads();
    for (int i = threadIdx.x; i < packs * rows; i += blockDim.x) {
      const int pack = i % packs, r = i / packs;
      float mean[VEC], m2[VEC];
      int have = 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) mean[v] = m2[v] = 0.f;
      const T* from = x + (long long)r * p.x_stride_t + pack * VEC;
      const long long step = (long long)rows * p.x_stride_t;
      // `more` tokens: their means, their squares around them, and both into what there is
      auto batch = [&](auto full, int more) {
        constexpr bool FULL = decltype(full)::value;
        Pack<T, VEC> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (FULL || u < more) raw[u] = load_pack<T, VEC>(from);
          else raw[u].zero();
          if (FULL || u < more) from += step;
        }
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
        const float inv = FULL ? 1.f / U : 1.f / (float)more, share = (float)more / (float)(have + more), weight = (float)have * share;
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] *= inv;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[VEC];
          raw[u].get(f);
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            if (FULL || u < more) sq[v] = fmaf(f[v] - sum[v], f[v] - sum[v], sq[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) join(mean[v], m2[v], sum[v], sq[v], share, weight);
        have += more;
      };
      int left = r < tokens ? (tokens - r + rows - 1) / rows : 0;
      for (; left >= U; left -= U) batch(std::true_type(), U);
      if (left > 0) batch(std::false_type(), left);
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (pack * VEC + v < chans) s_mean[r * chans + pack * VEC + v] = mean[v], s_m2[r * chans + pack * VEC + v] = m2[v];
    }
    __syncthreads();
    // a warp a group: channels and token rows, each of the values it has
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, span = min(C, chans);
    for (int g = warp; g < chans / span; g += blockDim.x / 32) {
      const float values = (float)tokens * (float)span, inv = tokens > 0 ? 1.f / values : 0.f;
      float mean = 0.f, m2 = 0.f;
      for (int r = 0, at = g * span; r < rows; ++r, at += chans) {
        const float have = (float)((tokens - r + rows - 1) / rows);
        float s = 0.f;
        for (int i = lane; i < span; i += 32) s += s_mean[at + i];
        mean = fmaf(s, have * inv, mean);
      }
#pragma unroll
      for (int m = 16; m; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
      for (int r = 0, at = g * span; r < rows; ++r, at += chans) {
        const float have = (float)((tokens - r + rows - 1) / rows);
        if (have <= 0.f) break;
        for (int i = lane; i < span; i += 32) {
          const float d = s_mean[at + i] - mean;
          m2 += fmaf(d * d, have, s_m2[at + i]);
        }
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

template <typename T, int VEC, bool SILU>
__global__ void __launch_bounds__(WIDE, VEC >= 4 ? 1 : 2) group_norm_apply_kernel(const lq_group_norm_problem p, const Tiles t) {
  constexpr int U = kInFlight<VEC>;
  __shared__ float s_mean[CHANNELS], s_inv[CHANNELS];  // of the CTA's groups
  const int C = p.D / p.groups, b = blockIdx.z, g0 = blockIdx.y * t.block, groups = min(t.block, p.groups - g0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_enter();
  const int n = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.T) : p.T;
  const int first = (int)min((long long)blockIdx.x * t.tokens, (long long)p.T), stop = (int)min((long long)first + t.tokens, (long long)p.T);
  // The sums of the CTA's groups from all tiles, a group a warp. Up to 128 tiles are four values a lane, on their way together
  const float inv_n = n > 0 ? 1.f / (float)n : 0.f;
  for (int g = warp; g < groups; g += blockDim.x / 32) {
    const float2* sums = t.sums + (size_t)b * t.count * p.groups + g0 + g;
    auto tokens_of = [&](int i) { return i < t.count ? (float)min(max(n - i * t.tokens, 0), t.tokens) : 0.f; };  // behind the last tile i tokens may pass 32 bits
    float mean = 0.f, m2 = 0.f;
    if (t.count <= 128) {
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = lane + 32 * k < t.count ? sums[(size_t)(lane + 32 * k) * p.groups] : make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (const float have = tokens_of(lane + 32 * k); have > 0.f) mean = fmaf(have * inv_n, v[k].x, mean);
#pragma unroll
      for (int m = 16; m; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (const float have = tokens_of(lane + 32 * k); have > 0.f) m2 += fmaf((v[k].x - mean) * (v[k].x - mean), have * (float)C, v[k].y);
    } else {
      for (int i = lane; i < t.count; i += 32)
        if (const float have = tokens_of(i); have > 0.f) mean = fmaf(have * inv_n, sums[(size_t)i * p.groups].x, mean);
#pragma unroll
      for (int m = 16; m; m >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, m);
      for (int i = lane; i < t.count; i += 32)
        if (const float have = tokens_of(i); have > 0.f) {
          const float2 s = sums[(size_t)i * p.groups];
          m2 += fmaf((s.x - mean) * (s.x - mean), have * (float)C, s.y);
        }
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, m);
    if (lane == 0) s_mean[g] = mean, s_inv[g] = inv_std(m2 / ((float)n * (float)C), p.eps);
  }
  __syncthreads();
  const int width = groups * C, packs = (width + VEC - 1) / VEC, rows = max((int)blockDim.x / packs, 1);
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.x_stride_b + (long long)g0 * C;
  const T* gate = p.gate ? reinterpret_cast<const T*>(p.gate) + b * p.gate_stride_b + (long long)g0 * C : nullptr;
  T* y = reinterpret_cast<T*>(p.y) + (long long)b * p.T * p.D + (long long)g0 * C;
  for (int i = threadIdx.x; i < packs * rows; i += blockDim.x) {
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
    const T* from = x + (long long)(first + r) * p.x_stride_t + pack * VEC;
    const T* gated = gate ? gate + (long long)(first + r) * p.gate_stride_t + pack * VEC : nullptr;
    T* to = y + (long long)(first + r) * p.D + pack * VEC;
    const long long step = (long long)rows * p.x_stride_t, gate_step = (long long)rows * p.gate_stride_t, y_step = (long long)rows * p.D;
    auto batch = [&](auto count) {
      constexpr int N = decltype(count)::value;
      Pack<T, VEC> raw[N], z[N];
#pragma unroll
      for (int u = 0; u < N; ++u, from += step) raw[u] = load_pack<T, VEC>(from);
      if (gated)
#pragma unroll
        for (int u = 0; u < N; ++u, gated += gate_step) z[u] = load_pack<T, VEC>(gated);
#pragma unroll
      for (int u = 0; u < N; ++u, to += y_step) {
        float f[VEC];
        raw[u].get(f);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          f[v] = fmaf(f[v] - mean[v], a[v], c[v]);
          if constexpr (SILU) f[v] = silu(f[v]);
        }
        if (gated) {
          float zf[VEC];
          z[u].get(zf);
#pragma unroll
          for (int v = 0; v < VEC; ++v) f[v] *= silu(zf[v]);
        }
        Pack<T, VEC> out;
        out.set(f);
        store_pack(to, out);
      }
    };
    const int inside = min(stop, n) - first - r;  // of this thread's tokens: those of the sequence, then zeros
    int left = inside > 0 ? (inside + rows - 1) / rows : 0, zeros = (max(stop - first - r, 0) + rows - 1) / rows - left;
    for (; left >= U; left -= U) batch(std::integral_constant<int, U>());
    if (U > 4 && (left & 4)) batch(std::integral_constant<int, 4>());
    if (left & 2) batch(std::integral_constant<int, 2>());
    if (left & 1) batch(std::integral_constant<int, 1>());
    Pack<T, VEC> none;
    none.zero();
    for (; zeros > 0; --zeros, to += y_step) store_pack(to, none);
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
// Tiles of tokens: two CTAs an SM, at least 16 tokens each
static Tiles tiles_of(const lq_group_norm_problem* p) {
  Tiles t = {};
  const int C = p->D / p->groups;
  t.block = C >= CHANNELS ? 1 : CHANNELS / C;
  if (t.block > p->groups) t.block = p->groups;
  t.blocks = (p->groups + t.block - 1) / t.block;
  const long long columns = (long long)p->B * t.blocks, room = 2ll * sm_count();
  long long count = columns > 0 ? room / columns : 1;  // one more would be a second round for a few
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
        // a thread for every pack of a row where that is possible, several rows where it takes fewer than 512
        const int width = t.block * C < CHANNELS ? t.block * C : CHANNELS, packs = (width + VEC - 1) / VEC;
        const int threads = packs <= 320 || packs > WIDE ? 512 : (packs + 31) / 32 * 32;
        cudaError_t e = launch(group_norm_sums_kernel<T, VEC>, grid, dim3(threads), 0, st, *p, t);
        if (e == cudaSuccess)
          e = p->silu ? launch(group_norm_apply_kernel<T, VEC, true>, grid, dim3(threads), 0, st, *p, t) : launch(group_norm_apply_kernel<T, VEC, false>, grid, dim3(threads), 0, st, *p, t);
        return done(e);
      }
      const int packs = C / VEC;
      if (packs > 128) {
        const long long items = (long long)p->B * p->groups;
        if (items > 0x7fffffffll) return fail(LQ_ERR_SHAPE, "group_norm: %lld groups", items);
        return done(launch(group_norm_wide_kernel<T, VEC>, dim3((unsigned)items), dim3(THREADS), 0, st, *p));
      }
      // the narrowest team that holds a group in registers
      auto rows = [&](auto kern, int team, int pp) {
        const int teams = THREADS / team, block = p->groups < teams ? p->groups : teams, together = teams / block, columns = (p->groups + block - 1) / block;
        if (columns > 65535) return fail(LQ_ERR_SHAPE, "group_norm: D=%d groups=%d", p->D, p->groups);
        int per_sm = 0;
        cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, THREADS, 0);
        if (e != cudaSuccess) return done(e);
        // as many CTAs as the GPU holds, each with whole rounds of rows on their way where there are that many
        const long long need = ((long long)p->B + together - 1) / together, room = ((long long)sm_count() * per_sm + columns - 1) / columns, u = 4 / pp;
        const long long rounds = (need + room * u - 1) / (room * u), ctas = need <= room ? need : (need + rounds * u - 1) / (rounds * u);
        return done(launch(kern, dim3((unsigned)ctas, columns), dim3(THREADS), 0, st, *p, block, together));
      };
      return packs <= 8    ? rows(group_norm_rows_kernel<T, VEC, 8, 1>, 8, 1)
             : packs <= 16 ? rows(group_norm_rows_kernel<T, VEC, 8, 2>, 8, 2)
             : packs <= 32 ? rows(group_norm_rows_kernel<T, VEC, 16, 2>, 16, 2)
             : packs <= 64 ? rows(group_norm_rows_kernel<T, VEC, 32, 2>, 32, 2)
                           : rows(group_norm_rows_kernel<T, VEC, 32, 4>, 32, 4);
    };
    if (access == 16) return with_vec(std::integral_constant<int, FULL>());
    if constexpr (WORD > 1)
      if (access == 4) return with_vec(std::integral_constant<int, WORD>());
    return with_vec(std::integral_constant<int, 1>());
  });
}
