// Low-rank adapters beside the INT8 product: what its kernels add to their outputs.
//
//   y[m,n] += sum_r t[m,r] b[l,n,r],   l = adapters[m],   t[m,r] = scaling[l] x_scale[m] sum_k x[m,k] a[l,r,k]      (lq_lora.cu)
//
// Few tokens (at most 16): the product's kernel makes the sum itself. More: a kernel of its own has left it in fp32 for the rows that have an
// adapter (`share`), so that it joins the shared sum before either is rounded to y's type.
#pragma once
#include "lq_layer.cuh"

namespace lq {

constexpr int kFewTokens = 16;  // of the product's kernel that makes the adapters' sum itself

struct Lora {
  int L, R, RP;        // adapters; their rank, a multiple of 8; the pitch of t, a multiple of 16, zero behind R
  int dtype;           // of b
  const void* b;       // [L,N,R]
  const int* adapters; // [M]: which adapter a token has; one outside 0..L-1 is none
  const float* t;      // [M,RP]; 16-bit outputs of more than kFewTokens tokens: as two bf16 pieces of four values each
  // More than kFewTokens tokens. fp32 outputs: y itself, rows of N values. Else blocks of 32 tokens x 4 channels, channels before tokens: where the
  // product's lanes have a token each they read whole lines (in rows a line is fetched twice: 16384 x 2560 -> 10576, rank 16, 674 us, 514)
  float* share;
  int blocks;          // of 4 channels; 0 for rows
  __device__ __forceinline__ float* share_at(int m, int n) const {  // n: a multiple of 4
    return share + ((((long long)(m >> 5) * blocks + (n >> 2)) << 5) + (m & 31)) * 4;
  }
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

}  // namespace lq
