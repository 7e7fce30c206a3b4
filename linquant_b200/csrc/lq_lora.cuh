// Low-rank adapters beside the INT8 product: what its kernels add to a tile of outputs.
//
//   y[m,n] += sum_r t[m,r] b[l,n,r],   l = adapters[m],   t[m,r] = scaling[l] x_scale[m] sum_k x[m,k] a[l,r,k]      (lq_lora.cu)
#pragma once
#include "lq_layer.cuh"

namespace lq {

struct Lora {
  int L, R, RP;        // adapters; their rank, a multiple of 8; the pitch of t, a multiple of 16, zero behind R
  int dtype;           // of b
  const void* b;       // [L,N,R]
  const int* adapters; // [M]: which adapter a token has; one outside 0..L-1 is none
  const float* t;      // [M,RP] fp32, or for each four values their bf16 roundings, then those of what is left (16-bit outputs of the tcgen05 kernel)
  __device__ __forceinline__ int of(int m) const {
    const int l = __ldg(adapters + m);
    return (unsigned)l < (unsigned)L ? l : -1;
  }
};

// b[r .. r + 3] of a row as fp32; r a multiple of 4
__device__ __forceinline__ void lora_row4(const Lora& q, long long row, int r, float (&x)[4]) {
  const long long at = row * q.R + r;
  if (q.dtype == LQ_F32) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(q.b) + at));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(q.b) + at));
    if (q.dtype == LQ_F16) {
      x[0] = Act<__half>::get(v.x, 0), x[1] = Act<__half>::get(v.x, 1), x[2] = Act<__half>::get(v.y, 0), x[3] = Act<__half>::get(v.y, 1);
    } else {
      x[0] = Act<__nv_bfloat16>::get(v.x, 0), x[1] = Act<__nv_bfloat16>::get(v.x, 1), x[2] = Act<__nv_bfloat16>::get(v.y, 0), x[3] = Act<__nv_bfloat16>::get(v.y, 1);
    }
  }
}

// A row of b on its way to L2
__device__ __forceinline__ void lora_prefetch(const Lora& q, long long row) {
  const int bytes = q.R * (q.dtype == LQ_F32 ? 4 : 2);
  const char* from = reinterpret_cast<const char*>(q.b) + row * bytes;
  for (int i = 0; i < bytes; i += 128) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(from + i));
}

// The sum of one output, in fp32
__device__ __forceinline__ float lora_dot(const Lora& q, int l, int N, int m, int n) {
  float s = 0.f;
  const float* t = q.t + (long long)m * q.RP;
  const long long row = (long long)l * N + n;
#pragma unroll 4
  for (int r = 0; r < q.R; r += 4) {
    float b[4];
    lora_row4(q, row, r, b);
    const float4 v = *reinterpret_cast<const float4*>(t + r);
    s = fmaf(v.x, b[0], s), s = fmaf(v.y, b[1], s), s = fmaf(v.z, b[2], s), s = fmaf(v.w, b[3], s);
  }
  return s;
}

// fp32 pairs as N pairs of bf16 pieces, the largest first
template <int N>
__device__ __forceinline__ void bf16_pieces(float a, float b, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = Act<__nv_bfloat16>::pack2(a, b);
    if (i + 1 < N) a -= __uint_as_float(p[i] << 16), b -= __uint_as_float(p[i] & 0xffff0000u);
  }
}

// The sums of 32 tokens (m0 + lane) and 8 NT channels, added to accumulator fragments: v[i][j] has the tokens 16 i + g (+ 8), the
// channels 8 j + 2 q (+ 1) from n0. One pass over R for each adapter that the tokens have, the operands of the next step requested before
// the products of this one. The reduction index is permuted alike in both operands: a lane takes four consecutive r. Both go in as
// PIECES bf16 pieces (b of bf16: one), products of pieces that add up to 8 PIECES bits or more behind the first are left out: 16
// bits for 16-bit outputs, 24 for fp32.
template <int NT, int PIECES>
struct LoraTile {
  const Lora& q;
  int N, n0 = 0, m0, mine, l = 0, r0 = 0;
  uint32_t all, rows = 0, left = 0;
  bool one;         // every token here has the same adapter
  uint32_t b[NT][4];  // two words of 16-bit values or four fp32
  uint4 t[2][2];
  __device__ __forceinline__ LoraTile(const Lora& q, int M, int N, int m0) : q(q), N(N), m0(m0) {
    const int lane = threadIdx.x & 31;
    mine = m0 + lane < M ? q.of(m0 + lane) : -1;
    all = __ballot_sync(0xffffffffu, mine >= 0);
    const int first = __shfl_sync(0xffffffffu, mine, 0);
    one = __all_sync(0xffffffffu, m0 + lane >= M || (mine >= 0 && mine == first));
  }
  // The rows of b for `width` channels from n, on their way to L2
  __device__ __forceinline__ void prefetch(int n, int width) const {
    const int lane = threadIdx.x & 31, size = q.dtype == LQ_F32 ? 4 : 2;
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    const bool first = mine >= 0 && (same & ((1u << lane) - 1)) == 0;  // an adapter's first token
    const char* from = reinterpret_cast<const char*>(q.b) + ((long long)mine * N + n) * q.R * size;
    if (first) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(from), "r"(min(width, N - n) * q.R * size) : "memory");
  }
  __device__ __forceinline__ void next_adapter() {
    l = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
    rows = __ballot_sync(0xffffffffu, mine == l);
    left &= ~rows;
    r0 = 0;
  }
  __device__ __forceinline__ void request() {
    const int lane = threadIdx.x & 31, g = lane >> 2, r = r0 + 4 * (lane & 3);
    const int rb = min(r, q.R - 4);  // behind R t is zero
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const long long at = ((long long)l * N + min(n0 + 8 * j + g, N - 1)) * q.R + rb;  // behind N nothing is stored
      if (q.dtype == LQ_F32) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(q.b) + at));
        b[j][0] = v.x, b[j][1] = v.y, b[j][2] = v.z, b[j][3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(q.b) + at));
        b[j][0] = v.x, b[j][1] = v.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * i + 8 * h + g;
        t[i][h] = make_uint4(0u, 0u, 0u, 0u);
        if (rows >> row & 1) t[i][h] = *reinterpret_cast<const uint4*>(q.t + (long long)(m0 + row) * q.RP + r);
      }
  }
  // the first operands for the channels from n
  __device__ __forceinline__ void begin(int n) {
    if (!all) return;
    n0 = n;
    left = all;
    next_adapter();
    request();
  }
  // the products of one step on `s`; the next step's operands are requested in between. False behind the adapter's last step
  __device__ __forceinline__ bool step(float (&s)[2][NT][4], bool& more) {
    uint32_t a[2][PIECES][4], w[NT][PIECES][2];
    const bool inside = r0 + 4 * ((int)threadIdx.x & 3) < q.R;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (PIECES == 2) {  // as the first kernel has left them
          a[i][0][h] = t[i][h].x, a[i][0][2 + h] = t[i][h].y, a[i][1][h] = t[i][h].z, a[i][1][2 + h] = t[i][h].w;
        } else {
          uint32_t lo[PIECES], hi[PIECES];
          bf16_pieces<PIECES>(__uint_as_float(t[i][h].x), __uint_as_float(t[i][h].y), lo);
          bf16_pieces<PIECES>(__uint_as_float(t[i][h].z), __uint_as_float(t[i][h].w), hi);
#pragma unroll
          for (int k = 0; k < PIECES; ++k) a[i][k][h] = lo[k], a[i][k][2 + h] = hi[k];
        }
      }
    if (q.dtype == LQ_BF16) {
#pragma unroll
      for (int j = 0; j < NT; ++j) w[j][0][0] = inside ? b[j][0] : 0u, w[j][0][1] = inside ? b[j][1] : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float x[4];
        if (q.dtype == LQ_F16) {
          x[0] = Act<__half>::get(b[j][0], 0), x[1] = Act<__half>::get(b[j][0], 1), x[2] = Act<__half>::get(b[j][1], 0), x[3] = Act<__half>::get(b[j][1], 1);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(b[j][e]);
        }
        uint32_t lo[PIECES], hi[PIECES];
        bf16_pieces<PIECES>(inside ? x[0] : 0.f, inside ? x[1] : 0.f, lo);
        bf16_pieces<PIECES>(inside ? x[2] : 0.f, inside ? x[3] : 0.f, hi);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) w[j][k][0] = lo[k], w[j][k][1] = hi[k];
      }
    }
    r0 += 16;
    const bool same = r0 < q.R;
    if (!same && (more = left != 0)) next_adapter();
    if (same || more) request();
#pragma unroll
    for (int k = PIECES - 1; k >= 0; --k) {
      if (k > 0 && q.dtype == LQ_BF16) continue;
#pragma unroll
      for (int o = PIECES - 1 - k; o >= 0; --o)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) mma_bf16(s[i][j], a[i][o][0], a[i][o][1], a[i][o][2], a[i][o][3], w[j][k][0], w[j][k][1]);
    }
    return same;
  }
  __device__ __forceinline__ void add(float (&v)[2][NT][4]) {
    if (!all) return;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    bool more = true;
    if (one) {
      while (step(v, more)) {}
      return;
    }
    while (more) {
      const uint32_t now = rows;
      float s[2][NT][4];  // apart from the outputs: an infinity or NaN in b is no other adapter's
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][j][e] = 0.f;
      while (step(s, more)) {}
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][j][e] += now >> (16 * i + g + 8 * (e >> 1)) & 1 ? s[i][j][e] : 0.f;
    }
  }
};

}  // namespace lq
