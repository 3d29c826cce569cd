// Beam search's selection: one pass over the logits (sum of exponentials and the nout best of
// each part of a row), then a merge per prompt.  The logits are read once: 64 x 8 rows of 131072 bf16
// (134 MB) take 51 us, 42 of them the pass at 3.2 TB/s, which is bound by instruction issue (51 % of
// the slots) and by barriers: an exponential, two conversions and two maxima a value.
//
// Precision: the exponentials are 2^x to 2^-22 of themselves, a thread's and a part's sums fp32, parts are joined
// and totals formed in 64 bits, (score + x) - lse.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nested_ssm.h"

namespace nssm_host {
int fail(int code, const char* fmt, ...);
}

namespace nssm {

constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kVecs = 4;                 // 16-byte pieces per thread and step
constexpr int kMaxOut = NSSM_MAX_BEAM_OUT;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
  int b, K, V, n, eos;
  int splits, steps;   // CTAs of a row, steps of kBeamThreads * kVecs pieces each
  const void* logits;
  int64_t l_b, l_k;
  const float* scores;
  const uint8_t* fin;
  float* out_s;
  int32_t* out_p;
  int32_t* out_t;
  uint8_t* out_f;
  float2* part;        // [b*K][splits]: max and sum of exp(x - max)
  uint64_t* cand;      // [b*K][splits][n]: keys, descending; 0 = none
};

// Candidates order by (logit, lower token): an order-preserving 32-bit image of the logit
// above the complement of the token.  -inf maps to 0x007fffff, so a key of a real candidate is
// never 0.
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // -0 and 0 are equal
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unorder32(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return ((uint64_t)order32(x) << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float ex2(float x) {   // 2^x, 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The nth (1-based) largest of the CTA's values (n <= kBeamThreads), by counting for each how many
// are larger or equal and earlier.
__device__ __forceinline__ uint64_t nth_of_block(uint64_t mine, int n, uint64_t* sh, uint64_t* result) {
  sh[threadIdx.x] = mine;
  __syncthreads();
  int rank = 0;
#pragma unroll 8
  for (int i = 0; i < kBeamThreads; i += 2) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sh + i);
    rank += (v.x > mine) + (v.y > mine);
    rank += (v.x == mine && i < (int)threadIdx.x) + (v.y == mine && i + 1 < (int)threadIdx.x);
  }
  if (rank == n - 1) *result = mine;
  __syncthreads();
  return *result;
}

// A lower bound of the nth largest of the CTA's values: the nth largest of a few of each warp's.  0
// where there are too few.
__device__ __forceinline__ uint32_t lower_bound_of_block(uint32_t mine, int n, uint64_t* sh, uint64_t* result) {
  const int t = min(32, (2 * n + kBeamWarps - 1) / kBeamWarps), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int k = 0; k < t; ++k) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) sh[warp * t + k] = top;
    const int who = __ffs(__ballot_sync(0xffffffffu, mine == top)) - 1;
    if (lane == who) mine = 0;
  }
  __syncthreads();
  const uint64_t v = tid < kBeamWarps * t ? sh[tid] : 0;
  int rank = 0;
  for (int i = 0; i < kBeamWarps * t; ++i) rank += sh[i] > v || (sh[i] == v && i < tid);
  if (tid < kBeamWarps * t && rank == n - 1) *result = v;
  __syncthreads();
  return (uint32_t)*result;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// The pieces of one step of one thread, as fp32 values (-inf outside the row and for what is not
// finite) with each piece's maximum.
template <bool BF16>
struct BeamRow {
  static constexpr int E = BF16 ? 8 : 4;                // elements of a 16-byte piece
  static constexpr int kStep = kBeamThreads * kVecs * E;
  static constexpr int es = BF16 ? 2 : 4;
  const char* base;
  int V, lead;    // pieces are 16-byte aligned in memory: piece 0 may begin `lead` elements before the row

  __device__ __forceinline__ int first(int step, int c) const {
    return step * kStep + (c * kBeamThreads + (int)threadIdx.x) * E - lead;
  }
  // a piece that crosses an end of the row, -inf outside
  static __device__ __noinline__ uint4 edge(const char* base, int V, int t0) {
    uint32_t w[4];
#pragma unroll 1
    for (int q = 0; q < 4; ++q) {
      uint32_t v = 0;
#pragma unroll 1
      for (int i = 0; i < E / 4; ++i) {
        const int t = t0 + q * (E / 4) + i;
        const bool in = t >= 0 && t < V;
        if constexpr (BF16)
          v |= (in ? (uint32_t) reinterpret_cast<const uint16_t*>(base)[t] : 0xff80u) << (16 * i);
        else
          v = in ? reinterpret_cast<const uint32_t*>(base)[t] : 0xff800000u;
      }
      w[q] = v;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void load(int t0, uint4& r) const {
    r = t0 >= 0 && t0 + E <= V ? __ldg(reinterpret_cast<const uint4*>(base + (int64_t)t0 * es)) : edge(base, V, t0);
  }
  __device__ __forceinline__ void fetch(int step, uint4* r) const {
#pragma unroll
    for (int c = 0; c < kVecs; ++c) load(first(step, c), r[c]);
  }
  // E values of a piece and the largest
  static __device__ __forceinline__ void values(const uint4& raw, float* x, float& mx) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (BF16) {
      __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        if (i) m2 = __hmax2_nan(m2, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      }
      mx = max_nan(__low2float(m2), __high2float(m2));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
      mx = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
    }
    if (!(mx <= 3.402823466e38f)) {              // NaN and +inf count as masked
      mx = kNegInf;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!(x[i] <= 3.402823466e38f)) x[i] = kNegInf;
        mx = fmaxf(mx, x[i]);
      }
    }
  }
  static __device__ __forceinline__ float unpack(const uint4* raw, float* x, float* mxc) {
#pragma unroll
    for (int c = 0; c < kVecs; ++c) values(raw[c], x + c * E, mxc[c]);
    return fmaxf(fmaxf(mxc[0], mxc[1]), fmaxf(mxc[2], mxc[3]));
  }
};

// The n best of list[0, total) to cur, sorted, by counting for each how many are larger.
__device__ __forceinline__ int rank_list(const uint64_t* list, int total, int n, uint64_t* cur) {
  for (int i = threadIdx.x; i < total; i += kBeamThreads) {
    const uint64_t k = list[i];
    int rank = 0;
    for (int j = 0; j < total; ++j) rank += list[j] > k;
    if (rank < n) cur[rank] = k;
  }
  __syncthreads();
  return min(total, n);
}

// The part again, exactly: each step's candidates are those above the nout-th largest of the
// threads' own best keys, at most nout threads' values.
template <bool BF16>
__device__ __noinline__ int beam_exact(BeamRow<BF16> r, int step0, int steps, int n, uint64_t* sh, uint64_t* list,
                                       uint64_t* cur, uint64_t* nth, int* count) {
  constexpr int E = BeamRow<BF16>::E;
  int have = 0;
  for (int st = step0; st < step0 + steps; ++st) {
    uint4 raw[kVecs];
    float x[kVecs * E], mxc[kVecs];
    r.fetch(st, raw);
    r.unpack(raw, x, mxc);
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kVecs * E; ++i) {
      const int tk = r.first(st, i / E) + i % E;
      const uint64_t k = tk >= 0 && tk < r.V ? key_of(x[i], tk) : 0;
      best = k > best ? k : best;
    }
    if (threadIdx.x == 0) *count = 0;
    const uint64_t least = nth_of_block(best, n, sh, nth);
    if (best >= least)
#pragma unroll
      for (int i = 0; i < kVecs * E; ++i) {
        const int tk = r.first(st, i / E) + i % E;
        if (tk >= 0 && tk < r.V && key_of(x[i], tk) >= least) list[atomicAdd(count, 1)] = key_of(x[i], tk);
      }
    __syncthreads();
    const int found = *count;
    for (int i = threadIdx.x; i < have; i += kBeamThreads) list[found + i] = cur[i];
    __syncthreads();
    have = rank_list(list, found + have, n, cur);
  }
  return have;
}

// A part of a row, a step of kBeamThreads * kVecs 16-byte pieces at a time, the next one's loads in
// flight; the max, the sum and the candidates of a step all come from one read into registers.
// Candidates are the values that reach a lower bound of the nout-th best, the nout-th best of a
// few maxima of each warp in the first step, so most steps need no barrier; a step only notes
// the pieces that hold any, which are read again and ranked after a few steps (the bound then rises)
// and at the end.  Where the bound lets through too many (sorted or constant logits), beam_exact
// reads the part again.
template <bool BF16>
__global__ void __launch_bounds__(kBeamThreads, BF16 ? 3 : 4) beam_scan_kernel(const BeamParams p) {
  using Row = BeamRow<BF16>;
  constexpr int E = Row::E;
  constexpr int kCap = kMaxOut * kVecs * E;             // beam_exact's candidates: kMaxOut threads' values
  constexpr int kPieces = 1024;
  __shared__ __align__(16) uint64_t sh[kBeamThreads];
  __shared__ uint64_t list[kCap + kMaxOut], cur[kMaxOut];
  __shared__ float red[kBeamWarps], rsum[kBeamWarps];
  __shared__ uint64_t nth;
  __shared__ int plist[kPieces];                        // first tokens of the pieces that reach the bound
  __shared__ int count, pieces;
  const int row = blockIdx.y, bi = row / p.K, ki = row - bi * p.K, split = blockIdx.x;
  if (p.fin && p.fin[row]) return;                      // the merge knows its one candidate
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Row r;
  r.base = static_cast<const char*>(p.logits) + (bi * p.l_b + ki * p.l_k) * Row::es;
  r.V = p.V;
  r.lead = (int)((reinterpret_cast<uintptr_t>(r.base) & 15) / Row::es);
  const int step0 = split * p.steps;
  const int steps = max(0, min(p.steps, (p.V + r.lead + Row::kStep - 1) / Row::kStep - step0));
  float m = kNegInf, sum = 0.0f;                        // this thread's running maximum and sum
  float tau = kNegInf;
  int have = 0;
  bool many = false;                                    // more candidates than the list is for
  if (tid == 0) count = pieces = 0;
  // the values of the noted pieces that reach the bound go to the list, read again; how many it has
  auto gather = [&]() {
    __syncthreads();
    const int np = pieces;
    if (np <= kPieces)
      for (int i = tid; i < np; i += kBeamThreads) {
        uint4 one;
        float v[E], top;
        r.load(plist[i], one);
        r.values(one, v, top);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int tk = plist[i] + e;
          if (v[e] >= tau && tk >= 0 && tk < p.V) {
            const int at = atomicAdd(&count, 1);
            if (at < kCap) list[at] = key_of(v[e], tk);
          }
        }
      }
    __syncthreads();
    const int found = np <= kPieces ? count : kCap + 1;
    __syncthreads();
    if (tid == 0) pieces = 0;
    return found;
  };
  // ranking is quadratic in the list: beyond this beam_exact's shorter lists are the cheaper way
  const int most = min(kCap, 256 + 6 * p.n);
  uint4 raw[kVecs];
  if (steps > 0) r.fetch(step0, raw);
  for (int st = step0; st < step0 + steps; ++st) {
    float x[kVecs * E], mxc[kVecs];
    const float mx = r.unpack(raw, x, mxc);
    if (st + 1 < step0 + steps) r.fetch(st + 1, raw);
    if (mx > m) {
      sum *= ex2((m - mx) * kLog2e);
      m = mx;
    }
    if (m != kNegInf) {
      // the difference first: x log2e - m log2e would leave the rounding of m log2e in every exponent, which for
      // logits of 1e9 and masks of -1e10 and beyond is a factor of up to infinity (one more instruction a
      // pair of values; 64 x 8 x 131072 take 51 us either way)
      float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      const float2 l2 = make_float2(kLog2e, kLog2e), off = make_float2(-m, -m);
#pragma unroll
      for (int i = 0; i < kVecs * E; i += 2) {
        const float2 e = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), off), l2);
        s2[(i >> 1) & 1] = __fadd2_rn(s2[(i >> 1) & 1], make_float2(ex2(e.x), ex2(e.y)));
      }
      sum += (s2[0].x + s2[0].y) + (s2[1].x + s2[1].y);
    }
    if (st == step0) {
      const uint32_t bound = lower_bound_of_block(order32(mx), p.n, sh, &nth);
      tau = unorder32(bound);
      if (!(tau >= kNegInf)) tau = kNegInf;     // fewer values than that
    }
    if (!many) {
#pragma unroll
      for (int c = 0; c < kVecs; ++c)
        if (mxc[c] >= tau) {
          const int at = atomicAdd(&pieces, 1);
          if (at < kPieces) plist[at] = r.first(st, c);
        }
      // after 3, 7, 15 .. steps the nout-th best so far becomes the bound, so that a long part does not
      // collect in proportion to its length
      const int done = st - step0 + 1;
      if (((done + 1) & done) == 0 && done > 2 && steps - done > 1) {
        const int found = gather();
        many = found > most;
        if (!many) {
          have = rank_list(list, found, p.n, cur);
          for (int i = tid; i < have; i += kBeamThreads) list[i] = cur[i];
          if (tid == 0) count = have;
          if (have == p.n) tau = unorder32((uint32_t)(cur[p.n - 1] >> 32));
          __syncthreads();
        }
      }
    }
  }
  if (!many) {
    const int found = gather();
    many = found > most;
    if (!many) have = rank_list(list, found, p.n, cur);
  }
  if (many) have = beam_exact<BF16>(r, step0, steps, p.n, sh, list, cur, &nth, &count);
  uint64_t* out = p.cand + ((int64_t)row * p.splits + split) * p.n;
  for (int i = tid; i < p.n; i += kBeamThreads) out[i] = i < have ? cur[i] : 0;
  // the part's maximum and sum
  float mm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (lane == 0) red[warp] = mm;
  __syncthreads();
  mm = red[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w) mm = fmaxf(mm, red[w]);
  if (mm != kNegInf) sum *= ex2((m - mm) * kLog2e);     // 0 for a thread without a value
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) rsum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    float s = 0.0f;
    for (int w = 0; w < kBeamWarps; ++w) s += rsum[w];
    p.part[(int64_t)row * p.splits + split] = make_float2(mm, s);
  }
}

// A candidate of the merge: its total, then the lower beam, then the beam's own order.
struct BeamKey {
  uint64_t hi;         // order-preserving image of the 64-bit total; 0 = none
  uint64_t lo;         // complement of the beam, logit order, complement of the token
  __device__ __forceinline__ bool operator<(const BeamKey& o) const { return hi < o.hi || (hi == o.hi && lo < o.lo); }
};
__device__ __forceinline__ uint64_t order64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double unorder64(uint64_t o) {
  return __longlong_as_double((long long)((o >> 63) ? (o & ~(1ull << 63)) : ~o));
}

constexpr int kBlock = 4 * kBeamThreads;     // candidates looked at together
constexpr int kBeamBits = 6, kTokenBits = 26;
static_assert(NSSM_MAX_BEAMS <= 1 << kBeamBits && kBeamBits + kTokenBits == 32, "fields of BeamKey::lo");

// One prompt: the nout best of all candidates.  The segments' lists are sorted, so candidates
// come in the order of their rank: the first block holds the heads of the lists, and once no list
// has anything above the nout-th best so far at some rank, nothing behind it has.
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamParams p) {
  __shared__ double lse[NSSM_MAX_BEAMS];
  __shared__ __align__(16) uint64_t sh[kBeamThreads];
  __shared__ BeamKey cur[kMaxOut], list[kBlock + kMaxOut];
  __shared__ uint64_t nth;
  __shared__ int count;
  const int bi = blockIdx.x, tid = threadIdx.x;
  for (int k = tid >> 5; k < p.K; k += kBeamThreads / 32) {   // a warp per beam
    const int64_t row = (int64_t)bi * p.K + k;
    const bool fin = p.fin && p.fin[row];
    float m = kNegInf;
    if (!fin)
      for (int s = tid & 31; s < p.splits; s += 32) m = fmaxf(m, p.part[row * p.splits + s].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double sum = 0.0;
    if (!fin && m != kNegInf)
      for (int s = tid & 31; s < p.splits; s += 32) {
        const float2 q = p.part[row * p.splits + s];
        if (q.x != kNegInf) sum += (double)q.y * exp((double)q.x - (double)m);
      }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) lse[k] = fin ? 0.0 : m == kNegInf ? (double)kNegInf : log(sum) + (double)m;
  }
  __syncthreads();
  const int lists = p.K * p.splits, per = min(p.n, p.V);
  const int64_t all = (int64_t)lists * per;
  int have = 0, quiet = 0;   // entries of cur; candidates since the last one that counted
  for (int64_t c0 = 0; c0 < all && quiet < lists; c0 += kBlock) {
    BeamKey key[4];
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      key[u] = BeamKey{0, 0};
      const int64_t c = c0 + u * kBeamThreads + tid;
      if (c >= all) continue;
      const int j = (int)(c / lists), l = (int)(c - (int64_t)j * lists), k = l / p.splits, split = l - k * p.splits;
      const int64_t row = (int64_t)bi * p.K + k;
      float x;
      uint32_t tok;
      if (p.fin && p.fin[row]) {
        if (split) continue;
        tok = j == 0 ? p.eos : j - 1 < p.eos ? j - 1 : j;
        x = j == 0 ? 0.0f : kNegInf;
      } else {
        const uint64_t q = p.cand[(row * p.splits + split) * p.n + j];
        if (!q) continue;
        tok = ~(uint32_t)q;
        x = unorder32((uint32_t)(q >> 32));
      }
      double total = ((double)p.scores[row] + (double)x) - lse[k];
      if (isnan(total)) total = (double)kNegInf;
      key[u].hi = order64(total);
      key[u].lo = ((uint64_t)((1 << kBeamBits) - 1 - k) << (32 + kTokenBits)) | ((uint64_t)order32(x) << kTokenBits) |
                  (~tok & ((1u << kTokenBits) - 1));
      best = key[u].hi > best ? key[u].hi : best;
    }
    if (tid == 0) count = 0;
    // at first a lower bound from the upper halves of the threads' best totals
    BeamKey tau{0, 0};
    if (c0 == 0)
      tau.hi = (uint64_t)lower_bound_of_block((uint32_t)(best >> 32), p.n, sh, &nth) << 32;
    else if (have == p.n)
      tau = cur[p.n - 1];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (key[u].hi && !(key[u] < tau)) list[atomicAdd(&count, 1)] = key[u];
    __syncthreads();
    const int found = count;
    if (found) {
      quiet = 0;
      for (int i = tid; i < have; i += kBeamThreads) list[found + i] = cur[i];
      __syncthreads();
      const int m = found + have;
      for (int i = tid; i < m; i += kBeamThreads) {
        const BeamKey k = list[i];
        int rank = 0;
        for (int j = 0; j < m; ++j) rank += k < list[j];
        if (rank < p.n) cur[rank] = k;
      }
      have = min(m, p.n);
    } else {
      quiet += kBlock;
    }
    __syncthreads();
  }
  for (int i = tid; i < p.n; i += kBeamThreads) {
    const BeamKey k = cur[i];
    const int beam = (1 << kBeamBits) - 1 - (int)(k.lo >> (32 + kTokenBits));
    const int tok = (int)(~(uint32_t)k.lo & ((1u << kTokenBits) - 1));
    const int64_t o = (int64_t)bi * p.n + i;
    p.out_s[o] = (float)unorder64(k.hi);
    p.out_p[o] = beam;
    p.out_t[o] = tok;
    if (p.out_f) p.out_f[o] = (tok == p.eos) || (p.fin && p.fin[(int64_t)bi * p.K + beam]);
  }
}

}  // namespace nssm

namespace {

using nssm_host::fail;

// CTAs of a row: about two waves of the call's CTAs over B200's 148 SMs (three of the bf16 pass fit on one,
// four of the fp32 pass), as few as that allows: a part's first step pays for the bound, and every part
// leaves nout candidates to the merge (64 x 8 rows of 131072, at an earlier step: 48 us with two waves, 54
// with four, 68 with six; 51 us now).  The workspace query, which needs no device, uses the same number.
void row_parts(int64_t rows, int V, int bf16, int* splits, int* steps) {
  const int per = nssm::kBeamThreads * nssm::kVecs * (bf16 ? 8 : 4);
  const int all = (int)(((int64_t)V + (bf16 ? 7 : 3) + per - 1) / per);   // a row may begin inside its first piece
  const int64_t want = (148 * 3 * 2 + rows - 1) / rows;
  *steps = want >= all ? 1 : (int)((all + want - 1) / want);
  *splits = (all + *steps - 1) / *steps;
}
size_t part_bytes(int64_t rows, int splits) { return ((size_t)rows * splits * sizeof(float2) + 255) / 256 * 256; }

}  // namespace

extern "C" {

size_t nssm_sizeof_beam_args(void) { return sizeof(nssm_beam_args); }

size_t nssm_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t nout, int32_t logits_dtype) {
  if (batch <= 0 || beams <= 0 || vocab <= 0 || nout <= 0) return 0;
  const int64_t rows = (int64_t)batch * beams;
  int splits, steps;
  row_parts(rows, vocab, logits_dtype == NSSM_BF16, &splits, &steps);
  return part_bytes(rows, splits) + (size_t)rows * splits * nout * sizeof(uint64_t);
}

int nssm_beam_select(const nssm_beam_args* a, void* stream) {
  if (!a) return fail(NSSM_ERR_INVALID, "args is NULL");
  if (a->batch < 0 || a->beams <= 0 || a->beams > NSSM_MAX_BEAMS)
    return fail(NSSM_ERR_INVALID, "batch %d, beams %d (1 to %d)", a->batch, a->beams, NSSM_MAX_BEAMS);
  if (a->vocab <= 0 || a->vocab > (1 << nssm::kTokenBits))
    return fail(NSSM_ERR_INVALID, "vocab %d outside [1, %d]", a->vocab, 1 << nssm::kTokenBits);
  if (a->nout <= 0 || a->nout > NSSM_MAX_BEAM_OUT || a->nout > (int64_t)a->beams * a->vocab)
    return fail(NSSM_ERR_INVALID, "nout %d outside [1, min(%d, beams * vocab)]", a->nout, NSSM_MAX_BEAM_OUT);
  if (a->logits_dtype != NSSM_F32 && a->logits_dtype != NSSM_BF16)
    return fail(NSSM_ERR_INVALID, "logits dtype must be F32 or BF16");
  if (a->eos_token >= a->vocab) return fail(NSSM_ERR_INVALID, "eos_token %d outside the vocabulary", a->eos_token);
  if (a->finished && a->eos_token < 0) return fail(NSSM_ERR_INVALID, "finished beams need an eos_token");
  const int64_t rows = (int64_t)a->batch * a->beams;
  if (rows > 65535) return fail(NSSM_ERR_INVALID, "batch * beams %lld beyond 65535", (long long)rows);
  if (a->batch == 0) return NSSM_OK;
  if (!a->logits || !a->scores || !a->out_scores || !a->out_parents || !a->out_tokens)
    return fail(NSSM_ERR_INVALID, "logits/scores/outputs must be non-NULL");
  const size_t need = nssm_beam_workspace_bytes(a->batch, a->beams, a->vocab, a->nout, a->logits_dtype);
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15) || a->workspace_bytes < need)
    return fail(NSSM_ERR_INVALID, "a 16-byte aligned workspace of %zu bytes is needed (got %zu)", need, a->workspace_bytes);
  nssm::BeamParams p{};
  p.b = a->batch; p.K = a->beams; p.V = a->vocab; p.n = a->nout; p.eos = a->eos_token;
  const int bf16 = a->logits_dtype == NSSM_BF16;
  row_parts(rows, p.V, bf16, &p.splits, &p.steps);
  p.logits = a->logits; p.l_b = a->logits_stride_b; p.l_k = a->logits_stride_k;
  p.scores = a->scores; p.fin = a->finished;
  p.out_s = a->out_scores; p.out_p = a->out_parents; p.out_t = a->out_tokens; p.out_f = a->out_finished;
  p.part = static_cast<float2*>(a->workspace);
  p.cand = reinterpret_cast<uint64_t*>(static_cast<char*>(a->workspace) + part_bytes(rows, p.splits));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(p.splits, (unsigned)rows);
  if (bf16)
    nssm::beam_scan_kernel<true><<<grid, nssm::kBeamThreads, 0, st>>>(p);
  else
    nssm::beam_scan_kernel<false><<<grid, nssm::kBeamThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(NSSM_ERR_CUDA, "beam_scan_kernel launch: %s", cudaGetErrorString(e));
  nssm::beam_merge_kernel<<<p.b, nssm::kBeamThreads, 0, st>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return fail(NSSM_ERR_CUDA, "beam_merge_kernel launch: %s", cudaGetErrorString(e));
  return NSSM_OK;
}

}  // extern "C"
