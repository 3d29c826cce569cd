// Moves of slots: copy / fork, clear, compaction and the reorder of beams.  One CTA turns the
// request into a list of moves whose sources no move writes (the plan), then every CTA copies
// pieces of that list.  Bound by HBM: each moved byte is read once and written once (512 beams of
// 3 layers, 350 MB moved: 102 us, 6.8 TB/s, a plain copy's speed).
#include <cuda_runtime.h>
#include <stdint.h>

#include "nested_ssm.h"

namespace nssm_host {
int fail(int code, const char* fmt, ...);
}

namespace nssm {

constexpr int kPlanThreads = 1024;
constexpr int kMaxRows = NSSM_MAX_SLOT_ROWS;
constexpr int kCopyThreads = 256;
constexpr int kPiece = 32768;                        // bytes of one copy work item
// Up to these sizes every CTA of the copy makes the plan itself: it costs less than a launch
constexpr int kFusedRows = 512, kFusedSlots = 16384;

enum : int { STATUS_BAD_SLOT_BIT = 1, STATUS_CONFLICT = NSSM_STATUS_CONFLICT };
enum : int { PLAN_COPY = 0, PLAN_CLEAR = 1, PLAN_REORDER = 2, PLAN_COMPACT = 3 };

struct PlanParams {
  int kind, n, S, pad, group;
  const int32_t* a;      // src, slots
  const int32_t* b;      // dst, parents
  int32_t* out;          // new_slots
  int* count;            // number of moves
  int2* list;            // (src, dst) of each
  int32_t* status;
};

// Exclusive prefix sum over the CTA of two counts packed in one word each; returns the totals.
template <int NT>
__device__ __forceinline__ int2 block_scan2(int2 v, int2* total, int2* warp_sums) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int yx = __shfl_up_sync(0xffffffffu, x.x, o), yy = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) { x.x += yx; x.y += yy; }
  }
  __syncthreads();
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  if (w == 0) {
    int2 s = lane < NT / 32 ? warp_sums[lane] : make_int2(0, 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int yx = __shfl_up_sync(0xffffffffu, s.x, o), yy = __shfl_up_sync(0xffffffffu, s.y, o);
      if (lane >= o) { s.x += yx; s.y += yy; }
    }
    if (lane < NT / 32) warp_sums[lane] = s;
  }
  __syncthreads();
  *total = warp_sums[NT / 32 - 1];
  const int2 base = w ? warp_sums[w - 1] : make_int2(0, 0);
  return make_int2(base.x + x.x - v.x, base.y + x.y - v.y);
}

__device__ __forceinline__ bool bit_set(uint32_t* m, int i) { return (m[i >> 5] >> (i & 31)) & 1u; }

// The moves of one request.  Dynamic shared memory: three bitmaps over the slots (slots read,
// slots written, slots written twice), for reorder and compact also two words per row.
// NT threads, kRowsPer consecutive rows each; `count` and `list` receive the moves, the CTA with
// `lead` also writes new_slots and the status.
template <int NT, int kRowsPer>
__device__ __forceinline__ void make_plan(const PlanParams& p, uint32_t* sm, int* count, int2* list, bool lead) {
  __shared__ int2 warp_sums[32];
  __shared__ int err;
  const int words = (p.S + 31) >> 5;
  uint32_t *rd = sm, *wr = sm + words, *wr2 = sm + 2 * words;
  int32_t* first = reinterpret_cast<int32_t*>(sm + 3 * words);   // reorder: first child; both: free slots
  int32_t* freed = first + p.n;
  for (int i = threadIdx.x; i < 3 * words; i += NT) sm[i] = 0;
  if (threadIdx.x == 0) err = 0;
  if (p.kind == PLAN_REORDER)
    for (int i = threadIdx.x; i < p.n; i += NT) first[i] = 0x7fffffff;
  __syncthreads();
  const int r0 = threadIdx.x * kRowsPer;
  int src[kRowsPer], dst[kRowsPer];   // -1: no move
  int bad = 0;
  int2 total;

  if (p.kind == PLAN_COPY || p.kind == PLAN_CLEAR) {
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      const int r = r0 + j;
      src[j] = dst[j] = -1;
      if (r >= p.n) continue;
      const int d = p.b[r], s = p.kind == PLAN_COPY ? p.a[r] : d;
      if (s == p.pad || d == p.pad) continue;
      if (s < 0 || s >= p.S || d < 0 || d >= p.S) { bad |= STATUS_BAD_SLOT_BIT; continue; }
      if (p.kind == PLAN_COPY && s == d) continue;
      src[j] = s; dst[j] = d;
    }
  } else if (p.kind == PLAN_REORDER) {
    int parent[kRowsPer];
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      const int r = r0 + j;
      parent[j] = -1;
      if (r >= p.n) continue;
      const int mine = p.a[r];      // slots that two rows name: wr2
      if (mine != p.pad && mine >= 0 && mine < p.S) {
        const uint32_t m = 1u << (mine & 31);
        if (atomicOr(&wr[mine >> 5], m) & m) {
          atomicOr(&wr2[mine >> 5], m);
          bad |= STATUS_CONFLICT;
        }
      }
      const int q = p.b[r], base = r / p.group * p.group;
      if (q < 0 || q >= min(p.group, p.n - base)) { bad |= STATUS_BAD_SLOT_BIT; continue; }
      const int s = p.a[base + q];
      if (s == p.pad) continue;
      if (s < 0 || s >= p.S) { bad |= STATUS_BAD_SLOT_BIT; continue; }
      parent[j] = base + q;
      atomicMin(&first[base + q], r);
    }
    __syncthreads();
    int2 cnt = make_int2(0, 0);   // x: children after the first, y: live rows without a child, in slots of their own
    bool extra[kRowsPer], free_row[kRowsPer];
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      const int r = r0 + j;
      extra[j] = parent[j] >= 0 && first[parent[j]] != r;
      const int s = r < p.n ? p.a[r] : p.pad;
      free_row[j] = r < p.n && s != p.pad && s >= 0 && s < p.S && first[r] == 0x7fffffff && !bit_set(wr2, s);
      cnt.x += extra[j]; cnt.y += free_row[j];
    }
    int2 at = block_scan2<NT>(cnt, &total, warp_sums);
    const int nfree = total.y;
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j)
      if (free_row[j]) freed[at.y++] = p.a[r0 + j];
    __syncthreads();
    for (int i = threadIdx.x; i < words; i += NT) wr[i] = wr2[i] = 0;
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      src[j] = dst[j] = -1;
      const int r = r0 + j;
      if (r >= p.n) continue;
      int s = parent[j] >= 0 ? p.a[parent[j]] : p.pad;
      if (extra[j]) {
        if (at.x < nfree) {
          src[j] = s;
          s = dst[j] = freed[at.x];
        } else {            // more children than slots: a row that is padded or shares its slot was to be continued
          bad |= STATUS_CONFLICT;
          s = p.pad;
        }
        ++at.x;
      }
      if (lead) p.out[r] = s;
    }
  } else {
    int2 cnt = make_int2(0, 0);   // x: live rows
    int slot[kRowsPer];
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      const int r = r0 + j;
      slot[j] = r < p.n ? p.a[r] : p.pad;
      if (slot[j] != p.pad && (slot[j] < 0 || slot[j] >= p.S)) { bad |= STATUS_BAD_SLOT_BIT; slot[j] = p.pad; }
      if (slot[j] != p.pad) {
        ++cnt.x;
        const uint32_t old = atomicOr(&rd[slot[j] >> 5], 1u << (slot[j] & 31));
        if (old & (1u << (slot[j] & 31))) bad |= STATUS_CONFLICT;
      }
    }
    block_scan2<NT>(cnt, &total, warp_sums);
    const int m = total.x;         // the live slots go to [0, m)
    cnt = make_int2(0, 0);         // x: rows that move, y: free slots below m
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      cnt.x += slot[j] != p.pad && slot[j] >= m;
      cnt.y += r0 + j < m && !bit_set(rd, r0 + j);
    }
    int2 at = block_scan2<NT>(cnt, &total, warp_sums);
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j)
      if (r0 + j < m && !bit_set(rd, r0 + j)) freed[at.y++] = r0 + j;
    __syncthreads();
    for (int i = threadIdx.x; i < words; i += NT) rd[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRowsPer; ++j) {
      src[j] = dst[j] = -1;
      if (r0 + j >= p.n) continue;
      if (slot[j] != p.pad && slot[j] >= m) {
        src[j] = slot[j];
        slot[j] = dst[j] = freed[at.x++];
      }
      if (lead) p.out[r0 + j] = slot[j];
    }
  }

  // drop moves into a slot that another move reads or writes (zeros may be written twice)
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kRowsPer; ++j)
    if (dst[j] >= 0 && p.kind != PLAN_CLEAR) {
      atomicOr(&rd[src[j] >> 5], 1u << (src[j] & 31));
      const uint32_t m = 1u << (dst[j] & 31);
      if (atomicOr(&wr[dst[j] >> 5], m) & m) atomicOr(&wr2[dst[j] >> 5], m);
    }
  __syncthreads();
  int2 cnt = make_int2(0, 0);
#pragma unroll
  for (int j = 0; j < kRowsPer; ++j)
    if (dst[j] >= 0) {
      if (bit_set(rd, dst[j]) || bit_set(wr2, dst[j])) {
        bad |= STATUS_CONFLICT;
        dst[j] = -1;
      } else {
        ++cnt.x;
      }
    }
  int2 at = block_scan2<NT>(cnt, &total, warp_sums);
#pragma unroll
  for (int j = 0; j < kRowsPer; ++j)
    if (dst[j] >= 0) list[at.x++] = make_int2(src[j], dst[j]);
  if (threadIdx.x == 0) *count = total.x;
  if (bad) atomicOr(&err, bad);
  __syncthreads();
  if (lead && threadIdx.x == 0 && err && p.status) atomicOr(p.status, err);
}

__global__ void __launch_bounds__(kPlanThreads) slot_plan_kernel(const PlanParams p) {
  extern __shared__ __align__(16) uint32_t sm[];
  make_plan<kPlanThreads, kMaxRows / kPlanThreads>(p, sm, p.count, p.list, true);
}

struct CopyBuffer {
  char* base;
  int64_t outer_stride, slot_stride, row_bytes;
  int per_row;     // pieces of one slot and layer
  int end;         // pieces of this buffer and those before it, per move
  int vec;         // 16, 4 or 1: the widest access that every row of the buffer allows
};
struct CopyParams {
  const int* count;
  const int2* list;
  int nbuf, clear;
  CopyBuffer buf[NSSM_MAX_SLOT_BUFFERS];
};

template <typename T>
__device__ __forceinline__ void copy_piece(char* dst, const char* src, int bytes, bool clear) {
  constexpr int kU = 8;
  const int n = bytes / (int)sizeof(T);
  const T* s = reinterpret_cast<const T*>(src);
  T* d = reinterpret_cast<T*>(dst);
  for (int i0 = threadIdx.x; i0 < n; i0 += kU * kCopyThreads) {
    T v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + u * kCopyThreads;
      if (clear)
        v[u] = T{};
      else if (i < n)
        v[u] = s[i];
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + u * kCopyThreads;
      if (i < n) d[i] = v[u];
    }
  }
}

__device__ __forceinline__ void copy_moves(const CopyParams& p, int count, const int2* list) {
  const int pieces = p.buf[p.nbuf - 1].end;
  const int64_t work = (int64_t)count * pieces;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int move = (int)(w / pieces);
    int piece = (int)(w - (int64_t)move * pieces), j = 0;
    while (piece >= p.buf[j].end) ++j;
    const CopyBuffer& b = p.buf[j];
    if (j) piece -= p.buf[j - 1].end;
    const int layer = piece / b.per_row;
    const int64_t off = (int64_t)(piece - layer * b.per_row) * kPiece;
    const int bytes = (int)min((int64_t)kPiece, b.row_bytes - off);
    const int2 m = list[move];
    const char* src = b.base + layer * b.outer_stride + m.x * b.slot_stride + off;
    char* dst = b.base + layer * b.outer_stride + m.y * b.slot_stride + off;
    if (b.vec == 16)
      copy_piece<int4>(dst, src, bytes, p.clear);
    else if (b.vec == 4)
      copy_piece<int32_t>(dst, src, bytes, p.clear);
    else
      copy_piece<char>(dst, src, bytes, p.clear);
  }
}

__global__ void __launch_bounds__(kCopyThreads) slot_copy_kernel(const CopyParams p) { copy_moves(p, *p.count, p.list); }

// Plan and copy in one launch.  Every CTA reads the request before it copies and none writes it
// (new_slots is another array, the leading CTA's alone).
__global__ void __launch_bounds__(kCopyThreads) slot_move_kernel(const PlanParams q, const CopyParams p) {
  extern __shared__ __align__(16) uint32_t sm[];
  __shared__ int2 list[kFusedRows];
  __shared__ int count;
  make_plan<kCopyThreads, kFusedRows / kCopyThreads>(q, sm, &count, list, blockIdx.x == 0);
  __syncthreads();
  copy_moves(p, count, list);
}

}  // namespace nssm

namespace {

using nssm_host::fail;

int check_buffers(const nssm_slot_buffer* bufs, int nbuf, int S, nssm::CopyParams& c) {
  if (!bufs || nbuf <= 0 || nbuf > NSSM_MAX_SLOT_BUFFERS)
    return fail(NSSM_ERR_INVALID, "%d slot buffers (1 to %d)", nbuf, NSSM_MAX_SLOT_BUFFERS);
  if (S <= 0 || S > NSSM_MAX_MOVE_SLOTS) return fail(NSSM_ERR_INVALID, "num_slots %d outside [1, %d]", S, NSSM_MAX_MOVE_SLOTS);
  int64_t end = 0;
  for (int i = 0; i < nbuf; ++i) {
    const nssm_slot_buffer& b = bufs[i];
    if (!b.base || b.outer <= 0 || b.row_bytes <= 0) return fail(NSSM_ERR_INVALID, "slot buffer %d is empty", i);
    if (b.slot_stride < b.row_bytes && S > 1) return fail(NSSM_ERR_INVALID, "slots of buffer %d overlap", i);
    if (b.outer > 1 && (b.outer_stride < 0 || (b.outer_stride < b.row_bytes)))
      return fail(NSSM_ERR_INVALID, "layers of buffer %d overlap", i);
    const int64_t per = (b.row_bytes + nssm::kPiece - 1) / nssm::kPiece;
    end += per * b.outer;
    if (end > (1 << 30)) return fail(NSSM_ERR_INVALID, "a slot of buffer %d is too large", i);
    const uint64_t a = reinterpret_cast<uintptr_t>(b.base) | (uint64_t)b.slot_stride | (uint64_t)b.row_bytes |
                       (b.outer > 1 ? (uint64_t)b.outer_stride : 0);
    c.buf[i] = {static_cast<char*>(b.base), b.outer > 1 ? b.outer_stride : 0, b.slot_stride, b.row_bytes, (int)per,
                (int)end, a % 16 == 0 ? 16 : a % 4 == 0 ? 4 : 1};
  }
  c.nbuf = nbuf;
  return NSSM_OK;
}

int move(nssm::PlanParams p, const nssm_slot_buffer* bufs, int nbuf, void* ws, size_t ws_bytes, void* stream) {
  if (p.n < 0 || p.n > NSSM_MAX_SLOT_ROWS) return fail(NSSM_ERR_INVALID, "rows %d outside [0, %d]", p.n, NSSM_MAX_SLOT_ROWS);
  nssm::CopyParams c{};
  int rc = check_buffers(bufs, nbuf, p.S, c);
  if (rc) return rc;
  if (p.n == 0) return NSSM_OK;
  const size_t need = nssm_slot_workspace_bytes(p.n);
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 7) || ws_bytes < need)
    return fail(NSSM_ERR_INVALID, "an 8-byte aligned workspace of %zu bytes is needed (got %zu)", need, ws_bytes);
  p.count = static_cast<int*>(ws);
  p.list = reinterpret_cast<int2*>(static_cast<char*>(ws) + 8);
  c.count = p.count;
  c.list = p.list;
  c.clear = p.kind == nssm::PLAN_CLEAR;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int dev = 0, sms = 0;
  // three bitmaps of the slots (48 KB at the most slots) and two words per row
  const int smem = 3 * ((p.S + 31) / 32) * 4 + 2 * p.n * 4;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool fused = p.n <= nssm::kFusedRows && p.S <= nssm::kFusedSlots;
  if (e == cudaSuccess && !fused && smem > 40 * 1024)
    e = cudaFuncSetAttribute(nssm::slot_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             3 * NSSM_MAX_MOVE_SLOTS / 8 + 2 * NSSM_MAX_SLOT_ROWS * 4);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(NSSM_ERR_CUDA, "slot moves: %s", cudaGetErrorString(e));
  }
  const int64_t work = (int64_t)p.n * c.buf[nbuf - 1].end;
  const int grid = (int)(work < 8 * sms ? work : 8 * sms);   // 2048 threads per SM
  if (fused) {
    nssm::slot_move_kernel<<<grid, nssm::kCopyThreads, smem, st>>>(p, c);
  } else {
    nssm::slot_plan_kernel<<<1, nssm::kPlanThreads, smem, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return fail(NSSM_ERR_CUDA, "slot_plan_kernel launch: %s", cudaGetErrorString(e));
    nssm::slot_copy_kernel<<<grid, nssm::kCopyThreads, 0, st>>>(c);
  }
  if ((e = cudaGetLastError()) != cudaSuccess) return fail(NSSM_ERR_CUDA, "slot move launch: %s", cudaGetErrorString(e));
  return NSSM_OK;
}

}  // namespace

extern "C" {

size_t nssm_sizeof_slot_buffer(void) { return sizeof(nssm_slot_buffer); }

size_t nssm_slot_workspace_bytes(int32_t rows) { return rows <= 0 ? 0 : 8 + (size_t)rows * 8; }

int nssm_slot_copy(const nssm_slot_buffer* bufs, int32_t nbuf, int32_t num_slots, const int32_t* src,
                   const int32_t* dst, int32_t rows, int32_t pad_slot_id, void* workspace, size_t workspace_bytes,
                   int32_t* status, void* stream) {
  if (rows > 0 && !dst) return fail(NSSM_ERR_INVALID, "dst is NULL");
  nssm::PlanParams p{};
  p.kind = src ? nssm::PLAN_COPY : nssm::PLAN_CLEAR;
  p.n = rows; p.S = num_slots; p.pad = pad_slot_id; p.group = 1;
  p.a = src; p.b = dst; p.status = status;
  return move(p, bufs, nbuf, workspace, workspace_bytes, stream);
}

int nssm_slot_reorder(const nssm_slot_buffer* bufs, int32_t nbuf, int32_t num_slots, const int32_t* slots,
                      const int32_t* parents, int32_t rows, int32_t group, int32_t pad_slot_id, int32_t* new_slots,
                      void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (rows > 0 && (!slots || !parents || !new_slots)) return fail(NSSM_ERR_INVALID, "slots/parents/new_slots must be non-NULL");
  if (rows > 0 && (group <= 0 || rows % group)) return fail(NSSM_ERR_INVALID, "rows %d are not whole groups of %d", rows, group);
  if (rows > 0 && new_slots == slots) return fail(NSSM_ERR_INVALID, "new_slots must not be slots");
  nssm::PlanParams p{};
  p.kind = nssm::PLAN_REORDER;
  p.n = rows; p.S = num_slots; p.pad = pad_slot_id; p.group = group;
  p.a = slots; p.b = parents; p.out = new_slots; p.status = status;
  return move(p, bufs, nbuf, workspace, workspace_bytes, stream);
}

int nssm_slot_compact(const nssm_slot_buffer* bufs, int32_t nbuf, int32_t num_slots, const int32_t* slots,
                      int32_t rows, int32_t pad_slot_id, int32_t* new_slots, void* workspace, size_t workspace_bytes,
                      int32_t* status, void* stream) {
  if (rows > 0 && (!slots || !new_slots)) return fail(NSSM_ERR_INVALID, "slots/new_slots must be non-NULL");
  if (rows > 0 && new_slots == slots) return fail(NSSM_ERR_INVALID, "new_slots must not be slots");
  nssm::PlanParams p{};
  p.kind = nssm::PLAN_COMPACT;
  p.n = rows; p.S = num_slots; p.pad = pad_slot_id; p.group = 1;
  p.a = slots; p.out = new_slots; p.status = status;
  return move(p, bufs, nbuf, workspace, workspace_bytes, stream);
}

}  // extern "C"
