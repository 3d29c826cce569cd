// The gated delta rule on states S[headdim][dstate] (fp32), per value head h:
//   S <- e^g S;  u = beta (v - S k);  S <- S + u k^T;  y = scale S q
// One decode token (delta_step_kernel); nssm_delta_chunk.cuh takes prompts.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "nested_ssm.h"

namespace nssm {

enum : int { STATUS_CONFLICT = NSSM_STATUS_CONFLICT };

struct DeltaStepParams {
  int H, G, P, S, ns, rows;   // ns slices of `rows` headdim rows per head
  int pad;
  int io_bf16, g_bf16, beta_bf16, out_bf16;
  int vec;                    // q and k rows are 8-byte (bf16) / 16-byte (fp32) aligned
  float scale;
  float* state;
  int64_t st_s;
  const void *q, *k, *v, *g, *beta;
  int64_t q_b, q_h, k_b, k_h, v_b, v_h, g_b, g_h, beta_b, beta_h;
  const int32_t* idx;
  void* out;
  int64_t o_b, o_h;
  int32_t* status;
};

__device__ __forceinline__ float dl_ld(const void* p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void dl_st(void* p, int64_t i, int bf16, float v) {
  if (bf16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    reinterpret_cast<float*>(p)[i] = v;
}
__device__ __forceinline__ float4 dl_ld4(const void* p, int64_t i, int bf16, int vec) {
  if (vec) {
    if (bf16) {
      const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
      return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                         __uint_as_float(r.y & 0xffff0000u));
    }
    return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
  }
  return make_float4(dl_ld(p, i, bf16), dl_ld(p, i + 1, bf16), dl_ld(p, i + 2, bf16), dl_ld(p, i + 3, bf16));
}
__device__ __forceinline__ float dot4(float4 a, float4 b, float acc) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, acc))));
}
// sum over the 4 lanes that share a state row
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// One decode token.  Bound by HBM: the state is read once and written once, 0.75 flop a byte.  A CTA
// takes `rows` state rows of one (batch row, head); 4 lanes share a state row, each with N/16 16-byte
// pieces of it in flight at once (128 bytes a thread at N = 128, which is what keeps HBM busy).  k and
// q of the head wait in shared memory.  The output is read off the old state,
// y = scale (e^g S q + u (k.q)), so that S k and S q reduce together.  448 rows of 128 heads of 80
// (4.7 GB): 782 to 823 us from box to box, 5.7 to 6.0 TB/s, with four CTAs of 40 rows an SM (one loads
// while another computes).  Timed on one box: 765 us so, 838 with two CTAs of 80 rows, 827 with five
// at 80 registers; 1883 with 8 lanes a row, half the bytes in flight and k and q in registers.  Rows are compared with the earlier rows' slots while the state is
// on its way.
constexpr int kStepRows = 40, kStepThreads = 4 * kStepRows;
template <int N>
__global__ void __launch_bounds__(kStepThreads, 4) delta_step_kernel(const DeltaStepParams p) {
  constexpr int V = N / 16;
  __shared__ float4 sk[N / 4], sq[N / 4];
  const int b = blockIdx.y, h = blockIdx.x / p.ns, slice = blockIdx.x - h * p.ns;
  const int tid = threadIdx.x, l4 = tid & 3;
  const int r = slice * p.rows + (tid >> 2);
  const int slot = p.idx ? p.idx[b] : b;
  if (slot == p.pad) return;
  if (slot < 0 || slot >= p.S) {
    if (p.status && blockIdx.x == 0 && tid == 0) atomicOr(p.status, 1);
    return;
  }
  const bool live = r < p.P;
  float4* row = reinterpret_cast<float4*>(p.state + (int64_t)slot * p.st_s + ((int64_t)h * p.P + (live ? r : 0)) * N) + l4;
  float4 s[V];
#pragma unroll
  for (int c = 0; c < V; ++c) s[c] = __ldcs(row + 4 * c);
  const int kh = h / (p.H / p.G);
  for (int i = tid; i < N / 2; i += blockDim.x) {
    const int n = i & (N / 4 - 1);
    if (i < N / 4)
      sk[n] = dl_ld4(p.k, b * p.k_b + kh * p.k_h + 4 * n, p.io_bf16, p.vec);
    else
      sq[n] = dl_ld4(p.q, b * p.q_b + kh * p.q_h + 4 * n, p.io_bf16, p.vec);
  }
  const float eg = expf(dl_ld(p.g, b * p.g_b + h * p.g_h, p.g_bf16));
  const float beta = dl_ld(p.beta, b * p.beta_b + h * p.beta_h, p.beta_bf16);
  const float v = live ? dl_ld(p.v, b * p.v_b + h * p.v_h + r, p.io_bf16) : 0.0f;
  // the first row that names a slot owns it
  int dup = 0;
  if (p.idx)
    for (int i = tid; i < b; i += blockDim.x) dup |= p.idx[i] == slot;
  if (__syncthreads_or(dup)) {
    if (p.status && blockIdx.x == 0 && tid == 0) atomicOr(p.status, STATUS_CONFLICT);
    return;
  }
  float ks = 0.0f, qs = 0.0f, kq = 0.0f;
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const float4 k4 = sk[l4 + 4 * c], q4 = sq[l4 + 4 * c];
    s[c].x *= eg; s[c].y *= eg; s[c].z *= eg; s[c].w *= eg;
    ks = dot4(s[c], k4, ks);
    qs = dot4(s[c], q4, qs);
    kq = dot4(k4, q4, kq);
  }
  ks = sum4(ks); qs = sum4(qs); kq = sum4(kq);
  const float u = beta * (v - ks);
  if (!live) return;
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const float4 k4 = sk[l4 + 4 * c];
    s[c].x = fmaf(u, k4.x, s[c].x); s[c].y = fmaf(u, k4.y, s[c].y);
    s[c].z = fmaf(u, k4.z, s[c].z); s[c].w = fmaf(u, k4.w, s[c].w);
    __stcs(row + 4 * c, s[c]);
  }
  if (l4 == 0) dl_st(p.out, b * p.o_b + h * p.o_h + r, p.out_bf16, p.scale * fmaf(u, kq, qs));
}

struct DeltaScanParams {
  int B, T, H, G, P;
  int g_bf16, beta_bf16;
  float scale;
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_b, q_t, k_b, k_t, v_b, v_t;
  const void *g, *beta;
  int64_t g_b, g_t, beta_b, beta_t;
  const int32_t* cu;
  const float* init;
  int64_t init_b;
  __nv_bfloat16* y;
  int64_t y_b, y_t;
  float* fin;
  int64_t fin_b;
  int32_t* status;
  uint32_t polls;        // limit of a bounded wait
};

// Tokens [t0, t0 + len) of sequence s (in its own batch row, or packed); false: bad bounds.
__device__ __forceinline__ bool delta_seq(const DeltaScanParams& p, int s, int* batch, int* t0, int* len) {
  if (!p.cu) {
    *batch = s; *t0 = 0; *len = p.T;
    return true;
  }
  const int a = p.cu[s], e = p.cu[s + 1];
  *batch = 0; *t0 = a; *len = e - a;
  return a >= 0 && e >= a && e <= p.T;
}

}  // namespace nssm
