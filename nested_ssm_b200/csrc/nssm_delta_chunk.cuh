// The gated delta rule over prompts in chunks of C tokens, on the tensor cores.
//
// With G_i the sum of g up to token i of a chunk, D_ij = e^{G_i - G_j} and S the state entering it:
//   A_ij = beta_i D_ij (k_i.k_j) for j < i,   T = (I + A)^-1,   M_ij = D_ij (q_i.k_j) for j <= i
//   r_i = beta_i (v_i - e^{G_i} S k_i),       u = T r
//   y_i = scale (e^{G_i} S q_i + sum_j M_ij u_j)
//   S  <- e^{G_C} S + sum_j e^{G_C - G_j} u_j k_j^T
// T and M do not depend on S: delta_prep_kernel computes them for every chunk in parallel and
// leaves them in the workspace as the B fragments of mma.m16n8k16.  delta_chunk_kernel then walks
// the chunks of a sequence.
//
// A warp owns 16 rows of S for the whole sequence, in the accumulator layout of m16n8k16, which is
// also that instruction's A layout: every product is taken in its transposed form (S K^T, R^T T^T,
// S Q^T, U^T M^T, U'^T K), so S, r and u go from one product to the next inside a warp's
// registers, and warps share only the K, Q, T and M tiles.  The chain of a chunk never leaves the
// register file; on tcgen05 each of its four dependent products would cross tensor memory twice,
// with the same conversions between (not built: with S transposed, dstate on the 128 lanes and the
// headdim as N, its rate is four times this one's).
//
// What bounds it.  Of 2 x 8192 tokens of 32 heads of 128 (551 us; input and output alone 63 us) the
// walk takes 442: a chain of 256 chunks, one warp on each quarter of 128 SMs, 1.73 us a chunk (3400
// cycles at 1965 MHz), of them 1170 cycles mma (146 products of 8 cycles a quarter) beside 660 of the
// helper warp with y (82 products).  Of 8 x 2048 tokens of 128 heads of 80 (1070 us; 128 us) it takes
// 880: two warps a quarter, 228 products a chunk, the tensor pipe 58 % busy (4 x 512 tokens), 4.3
// waves of CTAs.  Not kept (timed against 490 and 937 us, before y had two-piece operands): chunks of
// 64 with T by one substitution (four times the cost a chunk: 1703 us), bf16 operands in three pieces
// (316 products a chunk against 184; two pieces leave 3.6e-6 in the state), splitting the columns of S
// over two or four warps (the part of a chunk that is not split and the exchange take more than is won:
// 619 us), V by one small bulk copy a row (they cost the walk more than its arithmetic).
//
// Precision.  The state is fp32, and its products are to be as good: an fp32 operand goes in as two
// fp16 values (11 bits each, the second holds what the first leaves), scaled by a power of two that
// keeps the warp's values below 2^15; what is left out is below 2^-22 of a value or 2^-25.  K and Q
// (bf16) become fp16 exactly, each token scaled by its own power of two (elements below 2^-25 of the
// token's largest lose bits).  The r of a chunk share one scale, as do its u: those more than 2^17 below a warp's
// largest lose bits.  T, M and u go in as two pieces, so only products of two second pieces are
// left out, 2^-22 of a product.  y is the fp32 sum rounded once to bf16 (single fp16 operands, 2^-12, in its
// own products moved 3e-4 of it, and one value in thirty by a step; they take 504 against 551 us for 2 x 8192
// tokens of 32 heads, 950 against 1070 for 8 x 2048 of 128).
#pragma once

#include <cuda_fp16.h>

#include "nssm_delta.cuh"
#include "nssm_persistent.cuh"

namespace nssm {

constexpr int kC = 32;          // tokens of a chunk: a warp's lanes are its rows
constexpr int kTiles = kC / 8;
constexpr int kSteps = kC / 16;
// B fragments (32 lanes x 8 bytes) of a lower triangular 32 x 32 matrix: (nt, ks) holds token rows
// 8 nt.. and columns 16 ks..; those with ks <= nt / 2 exist
constexpr int kFrags = 6, kFragBytes = 256;
__host__ __device__ constexpr int frag_index(int nt, int ks) { return nt < 2 ? nt : 2 * nt - 2 + ks; }
// With k = sk k^ and q = sq q^ (sk, sq powers of two per token), the walk works on u~ = sk u.
// Where g > 0 lets a chunk's state grow, r, u and y of its tokens grow with it; each token then has a power of two c
// (1 while nothing has grown) that takes the growth since the smallest G out: with e^G' = c e^G and D' = e^{G'_i - G'_j}
// <= 1 in the place of e^G and D, the walk works on r~ = c r, u~ = sk c u and c y.
// Workspace block of a (chunk, head): two pieces of sT sk T, two of 2^-12 D' (q^.k^), then per token
// c beta, beta e^G' sk, 2^-12 e^G', 2^12 scale sq / c, e^{G_C - G'}, then 1 / sT, e^{G_C} and the larger of e^g of
// the first token and 1 (e^G' is not above it).
constexpr int kBlkM = 2 * kFrags * kFragBytes;
constexpr int kBlkF = kBlkM + 2 * kFrags * kFragBytes;
constexpr int kBlkBytes = kBlkF + 5 * kC * 4 + 32;    // whole sectors
// and of a (chunk, group): K^ and Q^ as the walk wants them in shared memory
template <int N> constexpr int kImgBytes = 2 * kC * N * 2;

struct DeltaChunkParams {
  DeltaScanParams s;
  unsigned char* img;    // [chunk][G][kImgBytes]
  unsigned char* blk;    // [chunk][H][kBlkBytes]
  int chunks;            // chunks of the workspace
  int per_seq;           // chunks of one sequence (not packed)
  int tiles;             // 16-row tiles of a head
  int tile_groups;       // CTAs per key group and sequence
  int heads;             // heads of a CTA's tiles at most
  int stages;            // chunks in shared memory
  int stuck;             // failure injection (tests only): CTA 0's first copies never complete
};

__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t hf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// Two fp32 values as two fp16 pairs that add up to them
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = hf2(a, b);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = hf2(a - f.x, b - f.y);
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Power-of-two scale that takes the largest of the warp's magnitudes m into [2^14, 2^15), and its
// inverse (m = 0, and m below 2^-112, count as 2^-112)
struct Pow2 { float s, inv; };
__device__ __forceinline__ Pow2 warp_scale(float m) {
  const uint32_t e = max(__reduce_max_sync(0xffffffffu, __float_as_uint(m)) >> 23, 15u);
  return {__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}
__device__ __forceinline__ float amax4(const float* v, float m) {
  return fmaxf(fmaxf(m, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void stsm4t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ uint32_t sm32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// A warp's bounded wait: one test that does not suspend (a phase that is over costs a fraction of a
// suspending try), then the tries; every lane observes the barrier.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t polls) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, ok)) return true;
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, polls));
}

// 16 bytes global -> shared, or zeros
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 32 bytes, a whole sector (two 16-byte stores would each write half of it)
__device__ __forceinline__ void st32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Byte offset of 16-byte piece c of row r in a [rows][N] bf16 tile: the pieces of 8 consecutive
// rows at one column lie in 8 different bank groups.
template <int N>
__device__ __forceinline__ uint32_t tile_off(int r, int c) { return (uint32_t)(r * (N * 2) + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ float ex2(float x) {   // 2^x, 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Chunks of sequence i, 0 where its bounds are bad.  Packed sequences take the workspace's chunks in their
// order, each behind those before it, so that no bounds let two sequences share one; a sequence for which there is
// no room (only sequences that overlap need more than there is) counts as bad.
__device__ __forceinline__ int seq_chunks(const DeltaScanParams& p, int i) {
  int batch, t0, len;
  return delta_seq(p, i, &batch, &t0, &len) ? (len + kC - 1) / kC : 0;
}

// ---------------------------------------------------------------- T and M of every chunk
// Bound by latency (a CTA loads, converts, multiplies, then solves) and by issue (58 %): 189 us for
// 8 x 2048 tokens of 128 heads, 109 for 2 x 8192 of 32 heads, which write 0.51 and 0.25 GB.  Seven CTAs
// an SM (with one piece of M: 170 and 104 us; with five CTAs 174 and 116, with four 178 and 128).
// CTA: one chunk and key group, 4 warps.  k.k and q.k come from the tensor cores once per group
// (products of bf16 values, fp32 sums); then a warp takes a head at a time, a lane a token row:
// row i of T solves T (I + A) = I from column i down in fp32 (a backward substitution over A's
// columns, read as broadcasts), and lies in the lane as the fragments want it.
constexpr int kPrepThreads = 128, kPrepWarps = kPrepThreads / 32;
constexpr int kPitch = kC + 4;    // floats: 16-byte reads of 8 lanes' rows fall into different banks

template <int N>
struct PrepSmem {
  // the columns of A (4 KB of each warp) take the place of the images once k.k and q.k are there
  static constexpr int kA = kPrepWarps * kC * kC * 4;
  static constexpr int off_kk = kImgBytes<N> > kA ? kImgBytes<N> : kA;
  static constexpr int off_qk = off_kk + kC * kPitch * 4;
  static constexpr int off_g = off_qk + kC * kPitch * 4;        // G as two floats, per warp
  static constexpr int off_s = off_g + kPrepWarps * 2 * kC * 4;    // sk, sq
  static constexpr int kBytes = off_s + 2 * kC * 4;
};

template <int N>
__global__ void __launch_bounds__(kPrepThreads, 7) delta_prep_kernel(const DeltaChunkParams p) {
  using L = PrepSmem<N>;
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ int s_seq, s_first;
  __shared__ int64_t s_sum[kPrepWarps];
  const int slot = blockIdx.x, grp = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int s = 0, first = 0;    // the sequence and its first chunk in the workspace
  if (!p.s.cu) {
    s = slot / p.per_seq;
    first = s * p.per_seq;
  } else {
    // each thread counts the chunks of a run of sequences; the one whose run has this chunk finds the sequence
    const int per = (p.s.B + kPrepThreads - 1) / kPrepThreads, i0 = min(tid * per, p.s.B), i1 = min(i0 + per, p.s.B);
    int64_t mine = 0;
    for (int i = i0; i < i1; ++i) mine += seq_chunks(p.s, i);
    int64_t to = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += y;
    }
    if (lane == 31) s_sum[warp] = to;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    for (int w = 0; w < warp; ++w) to += s_sum[w];
    if (to > slot && to - mine <= slot) {
      int at = (int)(to - mine);
      for (int i = i0;; ++i) {
        const int n = seq_chunks(p.s, i);
        if (slot < at + n) {
          s_seq = i;
          s_first = at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
    s = s_seq;
    if (s < 0) return;
    first = s_first;
  }
  int batch, t0, len;
  delta_seq(p.s, s, &batch, &t0, &len);
  const int c0 = (slot - first) * kC;
  const int nt = min(kC, len - c0);       // tokens of this chunk; the others count as zeros
  const int64_t tok = (int64_t)t0 + c0;
  const uint32_t sk = sm32(sm), sq = sk + kC * N * 2;
  unsigned char* img = p.img + ((int64_t)slot * p.s.G + grp) * kImgBytes<N>;
  float* ssk = reinterpret_cast<float*>(sm + L::off_s);
  // N / 8 neighbouring threads share a token: its largest exponent sets its scale
#pragma unroll
  for (int i = tid; i < kC * (N / 8); i += kPrepThreads) {
    const int r = i / (N / 8), c = i - r * (N / 8);
    uint4 kq[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (r < nt) {
      kq[0] = *reinterpret_cast<const uint4*>(p.s.k + batch * p.s.k_b + (tok + r) * p.s.k_t + grp * N + c * 8);
      kq[1] = *reinterpret_cast<const uint4*>(p.s.q + batch * p.s.q_b + (tok + r) * p.s.q_t + grp * N + c * 8);
    }
    const uint32_t o = tile_off<N>(r, c);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t w[4] = {kq[x].x, kq[x].y, kq[x].z, kq[x].w};
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) m = max(m, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
#pragma unroll
      for (int d = 1; d < N / 8; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
      // 2^e <= largest < 2^(e+1): times 2^(8-e)
      const uint32_t e = min(max(m >> 7, 16u), 250u);
      const float sc = __uint_as_float((262u - e) << 23);
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2) w[i2] = hf2(sc * bf_lo(w[i2]), sc * bf_hi(w[i2]));
      const uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(sm + x * kC * N * 2 + o) = v;
      *reinterpret_cast<uint4*>(img + x * kC * N * 2 + o) = v;
      if (c == 0) ssk[x * kC + r] = __uint_as_float((e - 8u) << 23);
    }
  }
  __syncthreads();
  float* kk = reinterpret_cast<float*>(sm + L::off_kk);
  float* qk = reinterpret_cast<float*>(sm + L::off_qk);
  {   // a warp: 16 rows of k.k or q.k against the columns up to their diagonal
    const int mt = warp >> 1, isq = warp & 1;
    float acc[kTiles][4] = {};
    const int row = mt * 16 + (lane & 15), half = lane >> 4;
#pragma unroll
    for (int ks = 0; ks < N / 16; ++ks) {
      uint32_t a[4];
      ldsm4(a, (isq ? sq : sk) + tile_off<N>(row, 2 * ks + half));
#pragma unroll
      for (int j = 0; j < kTiles; j += 2)
        if (j <= 2 * mt) {
          uint32_t b[4];   // two column tiles, two k halves each
          ldsm4(b, sk + tile_off<N>(8 * (j + (lane >> 4)) + (lane & 7), 2 * ks + ((lane >> 3) & 1)));
          mma16816(acc[j], a, b[0], b[1]);
          mma16816(acc[j + 1], a, b[2], b[3]);
        }
    }
    float* out = isq ? qk : kk;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; e += 2)
        *reinterpret_cast<float2*>(out + (mt * 16 + (lane >> 2) + 4 * e) * kPitch + 8 * j + (lane & 3) * 2) =
            make_float2(acc[j][e], acc[j][e + 1]);
  }
  __syncthreads();

  float* A = reinterpret_cast<float*>(sm) + warp * kC * kC;    // [column][row]
  float* gh = reinterpret_cast<float*>(sm + L::off_g) + warp * 2 * kC;
  float* gl = gh + kC;
  const int rep = p.s.H / p.s.G;
  // g and beta of this lane's token, a head ahead
  const int64_t og = batch * p.s.g_b + (tok + lane) * p.s.g_t, ob = batch * p.s.beta_b + (tok + lane) * p.s.beta_t;
  float ng = 0.0f, nbeta = 0.0f;
  auto fetch = [&](int hr) {
    if (lane < nt && hr < rep) {
      ng = dl_ld(p.s.g, og + grp * rep + hr, p.s.g_bf16);
      nbeta = dl_ld(p.s.beta, ob + grp * rep + hr, p.s.beta_bf16);
    }
  };
  fetch(warp);
  for (int hr = warp; hr < rep; hr += kPrepWarps) {
    const int h = grp * rep + hr;
    // G in units of ln 2: a 64-bit prefix sum, so that differences of far sums keep their
    // precision.  Below e^-104 a decay is zero in fp32: the clamp changes none and keeps -inf
    // out of the sums.
    double G = (ng < -120.0f ? -120.0 : (double)ng) * 1.4426950408889634;
    const float beta = nbeta;
    fetch(hr + kPrepWarps);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, G, o);
      if (lane >= o) G += y;
    }
    float low = (float)G;       // the smallest so far
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, low, o);
      if (lane >= o) low = fminf(low, y);
    }
    const int up = (int)fminf(ceilf((float)G - low), 126.0f);
    G -= (double)up;            // G'
    const float gih = (float)G, gil = (float)(G - (double)gih);
    gh[lane] = gih;
    gl[lane] = gil;
    __syncwarp();
    unsigned char* blk = p.blk + ((int64_t)slot * p.s.H + h) * kBlkBytes;
    float* f = reinterpret_cast<float*>(blk + kBlkF);
    const float c_inv = __uint_as_float((127 + up) << 23), up_end = (float)__shfl_sync(0xffffffffu, up, kC - 1);
    const float eg = ex2(gih + gil), ski = ssk[lane], bs = beta * ski;
    f[lane] = beta * __uint_as_float((127 - up) << 23);
    f[kC + lane] = bs * eg;
    f[2 * kC + lane] = eg * 0x1p-12f;
    f[3 * kC + lane] = p.s.scale * ssk[kC + lane] * 0x1p12f * c_inv;
    if (lane == kC - 1) f[5 * kC + 1] = ex2(gih + gil + up_end);
    if (lane == 0) f[5 * kC + 2] = fmaxf(eg, 1.0f);
    f[4 * kC + lane] = ex2((gh[kC - 1] - gih) + (gl[kC - 1] - gil) + up_end);
    // row `lane` of M, of A
    unsigned char* frow = blk + (lane & 7) * 32;      // its 32 bytes of each fragment
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      uint32_t mw[8], ml[8];
#pragma unroll
      for (int j = 16 * ks; j < 16 * ks + 16; j += 4) {
        const float4 h4 = *reinterpret_cast<const float4*>(gh + j), l4 = *reinterpret_cast<const float4*>(gl + j);
        const float4 k4 = *reinterpret_cast<const float4*>(kk + lane * kPitch + j);
        const float4 q4 = *reinterpret_cast<const float4*>(qk + lane * kPitch + j);
        const float4 s4 = *reinterpret_cast<const float4*>(ssk + j);
        const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
        const float hj[4] = {h4.x, h4.y, h4.z, h4.w}, lj[4] = {l4.x, l4.y, l4.z, l4.w};
        const float kj[4] = {k4.x, k4.y, k4.z, k4.w}, qj[4] = {q4.x, q4.y, q4.z, q4.w};
        float m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = ex2((gih - hj[e]) + (gil - lj[e]));
          m[e] = lane >= j + e ? d * (qj[e] * 0x1p-12f) : 0.0f;
          A[(j + e) * kC + lane] = lane > j + e ? bs * (sj[e] * (d * kj[e])) : 0.0f;
        }
        // columns c, c + 1 are lane (c & 7) / 2 of the fragment, columns c + 8, c + 9 its other word
        const int c = j & 15;
        split2(m[0], m[1], mw[(c & 7) + (c >> 3)], ml[(c & 7) + (c >> 3)]);
        split2(m[2], m[3], mw[(c & 7) + (c >> 3) + 2], ml[(c & 7) + (c >> 3) + 2]);
      }
      if (lane >= 16 * ks) {
        st32(frow + kBlkM + frag_index(lane >> 3, ks) * kFragBytes, mw);
        st32(frow + kBlkM + (kFrags + frag_index(lane >> 3, ks)) * kFragBytes, ml);
      }
    }
    __syncwarp();
    float x[kC];
#pragma unroll
    for (int j = kC - 1; j >= 0; --j) {
      float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = j / 4 * 4; k < kC; k += 4) {
        if (k + 3 <= j) continue;
        const float4 v = *reinterpret_cast<const float4*>(A + j * kC + k);
        if (k > j) a[0] = fmaf(v.x, x[k], a[0]);
        if (k + 1 > j) a[1] = fmaf(v.y, x[k + 1], a[1]);
        if (k + 2 > j) a[2] = fmaf(v.z, x[k + 2], a[2]);
        if (k + 3 > j) a[3] = fmaf(v.w, x[k + 3], a[3]);
      }
      x[j] = (j == lane ? 1.0f : 0.0f) - ((a[0] + a[1]) + (a[2] + a[3]));
    }
    float mx = 0.0f;
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      x[j] *= ski;
      mx = fmaxf(mx, fabsf(x[j]));
    }
    const Pow2 st = warp_scale(mx);
    if (lane == 0) f[5 * kC] = st.inv;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks)
      if (lane >= 16 * ks) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int c = 0; c < 16; c += 2)
          split2(st.s * x[16 * ks + c], st.s * x[16 * ks + c + 1], hi[(c & 7) + (c >> 3)], lo[(c & 7) + (c >> 3)]);
        st32(frow + frag_index(lane >> 3, ks) * kFragBytes, hi);
        st32(frow + (kFrags + frag_index(lane >> 3, ks)) * kFragBytes, lo);
      }
    __syncwarp();
  }
}

// ---------------------------------------------------------------- the walk over the chunks
// Chunks in shared memory.  Copies are issued (stages - 2) chunks ahead, into a stage that was in use
// two chunks ago: a chunk's copies take about as long as its work, and the warp that issues them
// should not wait for the slowest warp's last chunk.
constexpr int kChunkStages = 4;
constexpr int kSorted = 128;  // packed sequences that a CTA ranks by their length
constexpr int kWarps = 4;     // 16-row tiles of a CTA, one on each quarter of an SM
// A warp's own V tile: 32 tokens of 16 values, at a pitch that puts 8 rows into 8 bank groups; the
// next chunk's lies beside it.  y leaves through it.
constexpr int kVPitch = 48;
constexpr int kVBytes = kC * kVPitch;
template <int N>
struct ChunkSmem {
  static __host__ __device__ constexpr int stage(int heads) { return (kImgBytes<N> + heads * kBlkBytes + 127) / 128 * 128; }
  // what a tile's warp hands to its helper for a chunk: 16-column fragments of S's first pieces and of
  // its second ones, then those of u~ and two scales; two chunks, then the helper's y tile
  static constexpr int kHandU = 2 * (N / 16) * 512, kHandS = kHandU + 2 * kSteps * 512, kHand = kHandS + 16;
  static constexpr int kHelp = 2 * kHand + kVBytes;
  static __host__ __device__ constexpr int bytes(int stages, int heads, bool help) {
    return stages * stage(heads) + kWarps * (2 * kVBytes + (help ? kHelp : 0));
  }
};

// A CTA takes four consecutive tiles of the heads of one key group, which share K and Q; they may
// belong to different heads.  Two CTAs (up to 255 registers a thread) put two warps on each quarter
// of an SM, whatever the headdim (one CTA where it is 16 and dstate 128: four heads' T and M take
// 143 KB); three CTAs of 168 registers were slower (844 against 819 us for 8 x 2048 tokens of 128
// heads of 80, when those took 937 in all).
//
// HELP: where a call has no more CTAs than SMs, one warp on each quarter would do all of a chunk's
// work in turn.  y is not part of the chain from chunk to chunk, so a second warp computes it from
// the operands that the first one hands over (one prompt of 4096 tokens, 32 heads of
// 128, before y had two-piece operands: the walk 205 against 244 us).
template <int N, bool HELP>
__global__ void __launch_bounds__(kWarps * (HELP ? 64 : 32), HELP ? 1 : 2) delta_chunk_kernel(const DeltaChunkParams p) {
  using L = ChunkSmem<N>;
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ uint64_t full[kChunkStages], empty[kChunkStages], handed[kWarps][2], taken[kWarps][2];
  const int tid = threadIdx.x, lane = tid & 31, role = tid >> 5, warp = role % kWarps;   // warp: the tile in the CTA
  const bool helper = HELP && role >= kWarps;
  const int grp = blockIdx.x / p.tile_groups, tg = blockIdx.x - grp * p.tile_groups;
  int s = blockIdx.y, batch, t0, len;
  if (p.s.cu && p.s.B > 1 && p.s.B <= kSorted) {
    // the longest sequences first: CTAs start in this order, and the last ones to start should be short
    // (24 prompts of 35 to 700 tokens, 32 heads of 128, with one-piece operands of y: 206 against 231 us)
    __shared__ int lens[kSorted], chosen;
    for (int i = tid; i < p.s.B; i += blockDim.x) lens[i] = delta_seq(p.s, i, &batch, &t0, &len) ? len : 0;
    __syncthreads();
    for (int i = tid; i < p.s.B; i += blockDim.x) {
      int rank = 0;
      for (int j = 0; j < p.s.B; ++j) rank += lens[j] > lens[i] || (lens[j] == lens[i] && j < i);
      if (rank == (int)blockIdx.y) chosen = i;
    }
    __syncthreads();
    s = chosen;
  }
  if (!delta_seq(p.s, s, &batch, &t0, &len)) {
    if (p.s.status && blockIdx.x == 0 && tid == 0) atomicOr(p.s.status, STATUS_CONFLICT);
    return;
  }
  const int rep = p.s.H / p.s.G;
  const int warps = min(kWarps, rep * p.tiles - tg * kWarps);   // tiles that exist; the other warps only leave
  const int h0 = tg * kWarps / p.tiles;                         // first head of the CTA within the group
  const int nh = (tg * kWarps + warps - 1) / p.tiles - h0 + 1;
  const int hr = (tg * kWarps + warp) / p.tiles;                // the warp's
  const int h = grp * rep + hr, row_h = ((tg * kWarps + warp) - hr * p.tiles) * 16;
  const int nchunk = (len + kC - 1) / kC;
  __shared__ int64_t sums[2 * kWarps];      // chunks of the packed sequences before this one, by warps
  if (p.s.cu) {
    int64_t n = 0;
    for (int i = tid; i < s; i += blockDim.x) n += seq_chunks(p.s, i);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) sums[role] = n;
  }
  if (tid == 0) {
    for (int i = 0; i < kChunkStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], HELP ? 2 * warps : warps);
    }
    if (HELP)
      for (int i = 0; i < 2 * kWarps; ++i) {
        mbar_init(&handed[0][0] + i, 1);
        mbar_init(&taken[0][0] + i, 1);
      }
    fence_mbar_init();
  }
  __syncthreads();
  int64_t slot0 = (int64_t)s * p.per_seq;       // its first chunk in the workspace
  if (p.s.cu) {
    slot0 = 0;
    for (int w = 0; w < (HELP ? 2 : 1) * kWarps; ++w) slot0 += sums[w];
    if (nchunk && slot0 + nchunk > p.chunks) {
      if (p.s.status && blockIdx.x == 0 && tid == 0) atomicOr(p.s.status, STATUS_CONFLICT);
      return;
    }
  }
  if (warp >= warps) return;
  const uint32_t base = sm32(sm);
  const int stage = L::stage(p.heads), stages = p.stages, ahead = p.stages - 2;
  const __nv_bfloat16* gv = p.s.v + batch * p.s.v_b + (int64_t)t0 * p.s.v_t + h * p.s.P + row_h;
  const unsigned char* gimg = p.img + (slot0 * p.s.G + grp) * kImgBytes<N>;
  const unsigned char* gblk = p.blk + (slot0 * p.s.H + grp * rep + h0) * kBlkBytes;

  // K, Q, T and M of chunk c into its stage, by one warp
  auto load = [&](int c) {
    unsigned char* st = sm + (c % stages) * stage;
    uint64_t* bar = &full[c % stages];
    if (lane == 0) {
      const bool stuck = p.stuck && c == 0 && blockIdx.x == 0 && blockIdx.y == 0;
      mbar_expect_tx(bar, kImgBytes<N> + nh * kBlkBytes + (stuck ? 16 : 0));
      bulk_g2s(st, gimg + (int64_t)c * p.s.G * kImgBytes<N>, kImgBytes<N>, bar);
      bulk_g2s(st + kImgBytes<N>, gblk + (int64_t)c * p.s.H * kBlkBytes, nh * kBlkBytes, bar);
    }
    __syncwarp();
  };
  // the warp's V tile of chunk c, zeros for tokens that are not there
  const uint32_t vbase = base + stages * stage + warp * 2 * kVBytes;
  auto load_v = [&](int c) {
    const int nt = len - c * kC;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (lane >> 1) + 16 * i;
      cp16(vbase + (c & 1) * kVBytes + r * kVPitch + (lane & 1) * 16, gv + ((int64_t)c * kC + (r < nt ? r : 0)) * p.s.v_t + (lane & 1) * 8,
           r < nt);
    }
  };

  // y of chunk c, from O in the scale inv: through a tile in shared memory, then 16 bytes a lane
  auto finish = [&](float (*O)[4], const float* fac, float inv, uint32_t yt, int c) {
#pragma unroll
    for (int j = 0; j < kTiles; j += 2) {
      uint32_t w[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float2 k = *reinterpret_cast<const float2*>(fac + 3 * kC + 8 * (j + x) + (lane & 3) * 2);
        k.x *= inv;
        k.y *= inv;
        w[2 * x] = bf2(k.x * O[j + x][0], k.y * O[j + x][1]);
        w[2 * x + 1] = bf2(k.x * O[j + x][2], k.y * O[j + x][3]);
      }
      stsm4t(yt + (8 * (j + (lane >> 4)) + (lane & 7)) * kVPitch + ((lane >> 3) & 1) * 16, w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    const int nt = min(kC, len - c * kC);
    __nv_bfloat16* gy = p.s.y + batch * p.s.y_b + ((int64_t)t0 + (int64_t)c * kC) * p.s.y_t + h * p.s.P + row_h;
#pragma unroll
    for (int i = 0; i < kC / 16; ++i) {
      const int r = i * 16 + (lane >> 1), x = lane & 1;
      if (r < nt)
        *reinterpret_cast<uint4*>(gy + (int64_t)r * p.s.y_t + x * 8) =
            *reinterpret_cast<const uint4*>(sm + (yt - base) + r * kVPitch + x * 16);
    }
    __syncwarp();
  };
  // O += u M^T over 16 tokens, of two pieces each: first x first, first x second, second x first
  auto add_mu = [&](float (*O)[4], const uint32_t (*a)[4], const unsigned char* blk, int ks) {
    uint2 b[2][kTiles];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 2 * ks; j < kTiles; ++j)
        b[k][j] = *reinterpret_cast<const uint2*>(blk + lane * 8 + kBlkM + (k * kFrags + frag_index(j, ks)) * kFragBytes);
#pragma unroll
    for (int x = 0; x < 3; ++x)
#pragma unroll
      for (int j = 2 * ks; j < kTiles; ++j) mma16816(O[j], a[x >> 1], b[x & 1][j].x, b[x & 1][j].y);
  };
  auto hand_put = [&](unsigned char* at, const uint32_t* a) {
    *reinterpret_cast<uint4*>(at + lane * 16) = make_uint4(a[0], a[1], a[2], a[3]);
  };
  auto hand_get = [&](const unsigned char* at, uint32_t* a) {
    const uint4 q = *reinterpret_cast<const uint4*>(at + lane * 16);
    a[0] = q.x; a[1] = q.y; a[2] = q.z; a[3] = q.w;
  };
  unsigned char* hand = sm + stages * stage + kWarps * 2 * kVBytes + warp * L::kHelp;
  if constexpr (HELP) {
    if (helper) {
      bool ok = true;
      int si = 0, phase = 0;
      for (int c = 0; c < nchunk; ++c) {
        if (c && ++si == stages) {
          si = 0;
          phase ^= 1;
        }
        ok = warp_wait(&full[si], phase, p.s.polls);
        ok = ok && warp_wait(&handed[warp][c & 1], (c >> 1) & 1, p.s.polls);
        if (!ok) break;
        const uint32_t st = base + si * stage;
        const unsigned char* blk = sm + si * stage + kImgBytes<N> + (hr - h0) * kBlkBytes;
        const float* fac = reinterpret_cast<const float*>(blk + kBlkF);
        const unsigned char* in = hand + (c & 1) * L::kHand;
        float O[kTiles][4] = {};
#pragma unroll
        for (int ks = 0; ks < N / 16; ++ks) {
          uint32_t a[2][4], d[kTiles / 2][4];
#pragma unroll
          for (int x = 0; x < 2; ++x) hand_get(in + (x * (N / 16) + ks) * 512, a[x]);
#pragma unroll
          for (int j = 0; j < kTiles; j += 2)
            ldsm4(d[j / 2], st + kC * N * 2 + tile_off<N>(8 * (j + (lane >> 4)) + (lane & 7), 2 * ks + ((lane >> 3) & 1)));
#pragma unroll
          for (int x = 0; x < 2 * kTiles; ++x) {
            const int j = x % kTiles;
            mma16816(O[j], a[x / kTiles], d[j / 2][2 * (j & 1)], d[j / 2][2 * (j & 1) + 1]);
          }
        }
        const float2 sc = *reinterpret_cast<const float2*>(in + L::kHandS);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          float2 eg = *reinterpret_cast<const float2*>(fac + 2 * kC + 8 * j + (lane & 3) * 2);
          eg.x *= sc.x;
          eg.y *= sc.x;
#pragma unroll
          for (int e = 0; e < 4; ++e) O[j][e] *= e & 1 ? eg.y : eg.x;
        }
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          uint32_t a[2][4];
#pragma unroll
          for (int x = 0; x < 2; ++x) hand_get(in + L::kHandU + (2 * ks + x) * 512, a[x]);
          add_mu(O, a, blk, ks);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&taken[warp][c & 1]);
        finish(O, fac, sc.y, sm32(hand) + 2 * L::kHand, c);
        if (lane == 0) mbar_arrive(&empty[si]);
      }
      if (!ok && lane == 0 && p.s.status) atomicOr(p.s.status, STATUS_TIMEOUT);
      return;
    }
  }

  // S: tile t, element e: row lane / 4 + 8 (e / 2), column 8 t + 2 (lane % 4) + e % 2
  float S[N / 8][4];
  const int64_t row0 = ((int64_t)h * p.s.P + row_h + (lane >> 2)) * N + (lane & 3) * 2;
#pragma unroll
  for (int t = 0; t < N / 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float2 x = make_float2(0.0f, 0.0f);
      if (p.s.init) x = *reinterpret_cast<const float2*>(p.s.init + s * p.s.init_b + row0 + 8 * t + e * 4 * N);
      S[t][e] = x.x;
      S[t][e + 1] = x.y;
    }
  float m0 = 0.0f;
#pragma unroll
  for (int t = 0; t < N / 8; ++t) m0 = amax4(S[t], m0);
  Pow2 su{1.0f, 1.0f};        // the registers hold su.s S, no element of it above 2^15
  if (nchunk > 0) su = warp_scale(m0);
#pragma unroll
  for (int t = 0; t < N / 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[t][e] *= su.s;
  bool ok = true;
  if (warp == 0)
    for (int c = 0; c < min(ahead, nchunk); ++c) load(c);
  if (nchunk > 0) load_v(0);
  cp_commit();
  int turn = 0;         // the warp that issues the next copies
  int si = 0, phase = 0;                // the chunk's stage
  int last = min(ahead, nchunk) - 1;   // the last chunk whose copies this warp may have issued
  for (int c = 0; c < nchunk && ok; ++c) {
    const int next = c + ahead;
    if (warp == turn && next < nchunk) {
      // the stage is free once every warp is through the chunk that was in it
      if (next >= stages)
        ok = warp_wait(&empty[next % stages], (next / stages - 1) & 1, p.s.polls);
      if (ok) {
        load(next);
        last = next;
      }
    }
    turn = turn + 1 == warps ? 0 : turn + 1;
    if (c && ++si == stages) {
      si = 0;
      phase ^= 1;
    }
    if (c + 1 < nchunk) load_v(c + 1);
    cp_commit();
    cp_wait<1>();
    __syncwarp();      // every lane's part of V is there
    ok = warp_wait(&full[si], phase, p.s.polls) && ok;
    if (!ok) break;
    const uint32_t st = base + si * stage, vt = vbase + (c & 1) * kVBytes;
    const unsigned char* blk = sm + si * stage + kImgBytes<N> + (hr - h0) * kBlkBytes;
    const float* fac = reinterpret_cast<const float*>(blk + kBlkF);
    unsigned char* out = hand + (c & 1) * L::kHand;
    if (HELP && c >= 2) {     // the helper is through the chunk before the last
      ok = warp_wait(&taken[warp][c & 1], ((c >> 1) - 1) & 1, p.s.polls);
      if (!ok) break;
    }
    // P = S K^T and O = S Q^T (state rows x tokens)
    float Pm[kTiles][4] = {}, O[kTiles][4] = {};
    __half2 smax = __float2half2_rn(0.0f);
    uint32_t sa[2][2][4];     // pieces of 16 columns, of the next 16
    auto pieces = [&](int ks, int e) {
      split2(S[2 * ks + (e >> 1)][2 * (e & 1)], S[2 * ks + (e >> 1)][2 * (e & 1) + 1], sa[ks & 1][0][e], sa[ks & 1][1][e]);
      smax = __hmax2(smax, __habs2(*reinterpret_cast<__half2*>(&sa[ks & 1][0][e])));
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) pieces(0, e);
#pragma unroll
    for (int ks = 0; ks < N / 16; ++ks) {
      uint32_t b[kTiles / 2][4], d[kTiles / 2][4];
#pragma unroll
      for (int j = 0; j < kTiles; j += 2) {
        const uint32_t off = tile_off<N>(8 * (j + (lane >> 4)) + (lane & 7), 2 * ks + ((lane >> 3) & 1));
        ldsm4(b[j / 2], st + off);
        if (!HELP) ldsm4(d[j / 2], st + kC * N * 2 + off);
      }
      // products into one accumulator are apart by a round over the tiles; the next pieces between them
#pragma unroll
      for (int x = 0; x < 4 * kTiles; ++x) {
        const int j = x % kTiles, r = x / kTiles;
        if (r & 1) {
          if (!HELP) mma16816(O[j], sa[ks & 1][r / 2], d[j / 2][2 * (j & 1)], d[j / 2][2 * (j & 1) + 1]);
        } else {
          mma16816(Pm[j], sa[ks & 1][r / 2], b[j / 2][2 * (j & 1)], b[j / 2][2 * (j & 1) + 1]);
        }
        if (x % 4 == 0 && ks + 1 < N / 16) pieces(ks + 1, x / 4);
      }
      if (HELP)
#pragma unroll
        for (int x = 0; x < 2; ++x) hand_put(out + (x * (N / 16) + ks) * 512, sa[ks & 1][x]);
    }
    // r~ = c beta v - beta e^G' S k, in place
    float rmax = 0.0f;
#pragma unroll
    for (int j = 0; j < kTiles; j += 2) {
      uint32_t v[4];     // token tiles j, j + 1; rows 0-7 and 8-15 of each
      ldsm4t(v, vt + (8 * (j + (lane >> 4)) + (lane & 7)) * kVPitch + ((lane >> 3) & 1) * 16);
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const int t = 8 * (j + jj) + (lane & 3) * 2;
        const float2 be = *reinterpret_cast<const float2*>(fac + t);
        float2 bg = *reinterpret_cast<const float2*>(fac + kC + t);
        bg.x *= su.inv;
        bg.y *= su.inv;
        float* r = Pm[j + jj];
        r[0] = fmaf(-bg.x, r[0], be.x * bf_lo(v[2 * jj]));
        r[1] = fmaf(-bg.y, r[1], be.y * bf_hi(v[2 * jj]));
        r[2] = fmaf(-bg.x, r[2], be.x * bf_lo(v[2 * jj + 1]));
        r[3] = fmaf(-bg.y, r[3], be.y * bf_hi(v[2 * jj + 1]));
        rmax = amax4(r, rmax);
      }
    }
    const Pow2 fr = warp_scale(rmax);
    // U = R T~^T
    float U[kTiles][4] = {};
    const unsigned char* tf = blk + lane * 8;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      uint32_t a[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        split2(fr.s * Pm[2 * ks + (e >> 1)][2 * (e & 1)], fr.s * Pm[2 * ks + (e >> 1)][2 * (e & 1) + 1], a[0][e], a[1][e]);
      uint2 b[2][kTiles];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 2 * ks; j < kTiles; ++j)
          b[k][j] = *reinterpret_cast<const uint2*>(tf + (k * kFrags + frag_index(j, ks)) * kFragBytes);
#pragma unroll
      for (int x = 0; x < 3; ++x)     // first x first, first x second, second x first
#pragma unroll
        for (int j = 2 * ks; j < kTiles; ++j) mma16816(U[j], a[x >> 1], b[x & 1][j].x, b[x & 1][j].y);
    }
    // The scale of the state that follows: no element of it exceeds
    //   e^{G_C} max |S| + 32 max |k^| max |e^{G_C - G'} u~|,   |k^| < 512,
    // so its pieces can be taken from the registers as they are.  The bound may be 2^17 above the
    // state before its second pieces run into fp16's smallest values, and is seldom 2^10 above it.  (Where
    // every first piece is zero, |S| may be just below 2^-24.)
    // O has a scale of its own, so.s, with so.s |u~| below 2^15: a chunk may read a state and forget it that is far
    // above what it leaves.  Where S is more than 2^64 above u~, u~ loses bits instead of O leaving fp32.  No
    // factor between two scales leaves fp32: each scale is at most 2^104 above the largest of what it is applied to.
    const float inv_u = fr.inv * fac[5 * kC];
    float umax = 0.0f, wmax = 0.0f;
    float2 et[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      et[j] = *reinterpret_cast<const float2*>(fac + 4 * kC + 8 * j + (lane & 3) * 2);
      const float x = fmaxf(fabsf(U[j][0]), fabsf(U[j][2])), y = fmaxf(fabsf(U[j][1]), fabsf(U[j][3]));
      umax = fmaxf(umax, fmaxf(x, y));
      wmax = fmaxf(wmax, fmaxf(et[j].x * x, et[j].y * y));
    }
    const float egc = fac[5 * kC + 1];
    const float bs = su.inv * fmaxf(fmaxf(__low2float(smax), __high2float(smax)), 0x1p-24f);
    const float bu = inv_u * fmaxf(umax, 0x1p-24f);
    const Pow2 sn = warp_scale(fmaxf(2.001f * egc * bs, 0x1p15f * fmaxf(inv_u * wmax, 0x1p-64f * bu)));
    const Pow2 so = warp_scale(fmaxf(0x1p-64f * fac[5 * kC + 2] * bs, bu));
    const float os = su.inv * so.s, uo = inv_u * so.s, us = inv_u * sn.s, es = egc * su.inv * sn.s;
    su = sn;
#pragma unroll
    for (int t = 0; t < N / 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[t][e] *= es;
    // O = so.s (2^-12 e^G' S q^ + M u~)
    if (!HELP)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      float2 eg = *reinterpret_cast<const float2*>(fac + 2 * kC + 8 * j + (lane & 3) * 2);
      eg.x *= os;
      eg.y *= os;
#pragma unroll
      for (int e = 0; e < 4; ++e) O[j][e] *= e & 1 ? eg.y : eg.x;
    }
    // O += U M^T;  S += U' K
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      uint32_t a[2][4], au[2][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 ej = et[2 * ks + (e >> 1)];
        const float x = U[2 * ks + (e >> 1)][2 * (e & 1)], y = U[2 * ks + (e >> 1)][2 * (e & 1) + 1];
        split2(uo * x, uo * y, a[0][e], a[1][e]);
        split2(us * (ej.x * x), us * (ej.y * y), au[0][e], au[1][e]);
      }
      if (HELP) {
#pragma unroll
        for (int x = 0; x < 2; ++x) hand_put(out + L::kHandU + (2 * ks + x) * 512, a[x]);
      } else {
        add_mu(O, a, blk, ks);
      }
      if (HELP && ks == kSteps - 1) {
        if (lane == 0) *reinterpret_cast<float2*>(out + L::kHandS) = make_float2(os, so.inv);
        __syncwarp();
        if (lane == 0) mbar_arrive(&handed[warp][c & 1]);
      }
#pragma unroll
      for (int t = 0; t < N / 8; t += 4) {
        uint32_t b[2][4];   // column tiles t .. t + 3; token halves of each
#pragma unroll
        for (int x = 0; x < 2; ++x)
          ldsm4t(b[x], st + tile_off<N>(16 * ks + ((lane >> 3) & 1) * 8 + (lane & 7), t + 2 * x + (lane >> 4)));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) mma16816(S[t + x], au[i], b[x / 2][2 * (x & 1)], b[x / 2][2 * (x & 1) + 1]);
      }
    }
    if (!HELP) finish(O, fac, so.inv, vt, c);
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[si]);
  }
  if (!ok) {
    // a wait ran out: this warp's copies still in flight land (bounded) before it leaves
    if (lane == 0 && p.s.status) atomicOr(p.s.status, STATUS_TIMEOUT);
    cp_wait<0>();
    for (int c = max(0, last - ahead); c <= last; ++c)
      if ((c < ahead ? 0 : (c - ahead) % warps) == warp) mbar_wait_bounded(&full[c % stages], (c / stages) & 1, p.s.polls);
    return;
  }
  if (p.s.fin)
#pragma unroll
    for (int t = 0; t < N / 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; e += 2)
        *reinterpret_cast<float2*>(p.s.fin + s * p.s.fin_b + row0 + 8 * t + e * 4 * N) = make_float2(su.inv * S[t][e], su.inv * S[t][e + 1]);
}

}  // namespace nssm
