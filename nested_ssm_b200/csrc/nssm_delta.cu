// nssm_delta_step / nssm_delta_scan: argument checks and launches of the gated delta rule.
#include <cuda_runtime.h>
#include <math.h>
#include <stdlib.h>

#include "nssm_delta_chunk.cuh"

namespace nssm_host {
int fail(int code, const char* fmt, ...);
uint32_t wait_polls();   // nssm_set_wait_polls
int inject_stuck();      // nssm_test_inject_stuck_copy
}

namespace {

using nssm_host::fail;

bool al(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(n - 1)) == 0; }
bool io_ok(int d) { return d == NSSM_F32 || d == NSSM_BF16; }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NSSM_OK : fail(NSSM_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

int check_dims(int H, int G, int P, int N) {
  if (H <= 0 || G <= 0 || H % G || H > 8192) return fail(NSSM_ERR_INVALID, "nheads %d / ngroups %d", H, G);
  if (N != 64 && N != 128) return fail(NSSM_ERR_UNSUPPORTED, "dstate %d not compiled (supported: 64, 128)", N);
  if (P <= 0 || P % 16 || P > 256)
    return fail(NSSM_ERR_UNSUPPORTED, "headdim %d not supported (a multiple of 16 up to 256)", P);
  return NSSM_OK;
}

// State rows of one head over CTAs of 4 threads a row: at most 40 rows, and 16 where the whole
// call would otherwise not give every one of B200's 148 SMs two CTAs (one row of 32 heads of 128: 2.8 us either way; 448
// rows of 128 heads: 765 against 792 us).
void slices(int P, int64_t heads, int* ns, int* rows) {
  *ns = (P + nssm::kStepRows - 1) / nssm::kStepRows;
  *rows = ((P + *ns - 1) / *ns + 7) / 8 * 8;
  if (heads * *ns < 2 * 148) {
    *ns = P / 16;
    *rows = 16;
  }
}

using nssm::kC;

// Workspace chunks: of each sequence its own.  Packed sequences that do not overlap take
// sum ceil(len / C) <= seqlen / C + batch.
int64_t ws_chunks(int batch, int seqlen, int packed) {
  return packed ? (int64_t)seqlen / kC + batch : (int64_t)batch * ((seqlen + kC - 1) / kC);
}

constexpr int kMaxSmem = 227 * 1024 - 1024;    // of a walking CTA, beside its static 1 KB

template <int N>
int launch_chunks(nssm::DeltaChunkParams& p, void* ws, cudaStream_t st) {
  using L = nssm::ChunkSmem<N>;
  auto prep = nssm::delta_prep_kernel<N>;
  p.img = static_cast<unsigned char*>(ws);
  p.blk = p.img + (int64_t)p.chunks * p.s.G * nssm::kImgBytes<N>;
  const dim3 grid(p.s.G * p.tile_groups, p.s.B);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool help = (int64_t)grid.x * grid.y <= sms;
  auto walk = help ? nssm::delta_chunk_kernel<N, true> : nssm::delta_chunk_kernel<N, false>;
  p.stages = p.heads == 1 || (help && p.heads == 2) ? 4 : 3;   // as many as the CTAs of an SM have room for
  const int smem = L::bytes(p.stages, p.heads, help);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(prep, cudaFuncAttributeMaxDynamicSharedMemorySize, nssm::PrepSmem<N>::kBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(walk, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(walk, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  static_assert(L::bytes(4, 2, true) <= kMaxSmem && L::bytes(3, nssm::kWarps, true) <= kMaxSmem, "shared memory");
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(NSSM_ERR_CUDA, "delta scan: %s", cudaGetErrorString(e));
  }
  if (p.chunks > 0) {
    prep<<<dim3(p.chunks, p.s.G), nssm::kPrepThreads, nssm::PrepSmem<N>::kBytes, st>>>(p);
    const int rc = launched("delta_prep_kernel");
    if (rc) return rc;
  }
  walk<<<grid, nssm::kWarps * (help ? 64 : 32), smem, st>>>(p);
  return launched("delta_chunk_kernel");
}

}  // namespace

extern "C" {

size_t nssm_sizeof_delta_step_args(void) { return sizeof(nssm_delta_step_args); }
size_t nssm_sizeof_delta_scan_args(void) { return sizeof(nssm_delta_scan_args); }

int nssm_delta_step(const nssm_delta_step_args* a, void* stream) {
  if (!a) return fail(NSSM_ERR_INVALID, "args is NULL");
  if (a->batch < 0 || a->batch > 65535) return fail(NSSM_ERR_INVALID, "batch %d outside [0, 65535]", a->batch);
  if (a->num_slots <= 0) return fail(NSSM_ERR_INVALID, "num_slots %d", a->num_slots);
  int rc = check_dims(a->nheads, a->ngroups, a->headdim, a->dstate);
  if (rc) return rc;
  if (!io_ok(a->io_dtype) || !io_ok(a->g_dtype) || !io_ok(a->beta_dtype) || !io_ok(a->out_dtype))
    return fail(NSSM_ERR_INVALID, "io / g / beta / out dtype must be F32 or BF16");
  if (a->batch == 0) return NSSM_OK;
  if (!a->state || !a->q || !a->k || !a->v || !a->g || !a->beta || !a->out)
    return fail(NSSM_ERR_INVALID, "state/q/k/v/g/beta/out must be non-NULL");
  if (!a->state_batch_indices && a->batch > a->num_slots)
    return fail(NSSM_ERR_INVALID, "batch %d exceeds %d slots", a->batch, a->num_slots);
  if (!al(a->state, 16) || (a->state_stride_s & 3)) return fail(NSSM_ERR_INVALID, "state must be 16-byte aligned");
  if (a->state_stride_s < (int64_t)a->nheads * a->headdim * a->dstate)
    return fail(NSSM_ERR_INVALID, "state_stride_s smaller than a slot");
  if ((a->batch > 1 && llabs(a->out_stride_b) < a->headdim) || (a->nheads > 1 && llabs(a->out_stride_h) < a->headdim))
    return fail(NSSM_ERR_INVALID, "rows of out share memory");
  nssm::DeltaStepParams p{};
  p.H = a->nheads; p.G = a->ngroups; p.P = a->headdim; p.S = a->num_slots;
  slices(p.P, (int64_t)a->batch * p.H, &p.ns, &p.rows);
  p.pad = a->pad_slot_id;
  p.io_bf16 = a->io_dtype == NSSM_BF16; p.g_bf16 = a->g_dtype == NSSM_BF16;
  p.beta_bf16 = a->beta_dtype == NSSM_BF16; p.out_bf16 = a->out_dtype == NSSM_BF16;
  p.vec = al(a->q, p.io_bf16 ? 8 : 16) && al(a->k, p.io_bf16 ? 8 : 16) &&
          !((a->q_stride_b | a->q_stride_h | a->k_stride_b | a->k_stride_h) & 3);
  p.scale = a->scale;
  p.state = a->state; p.st_s = a->state_stride_s;
  p.q = a->q; p.q_b = a->q_stride_b; p.q_h = a->q_stride_h;
  p.k = a->k; p.k_b = a->k_stride_b; p.k_h = a->k_stride_h;
  p.v = a->v; p.v_b = a->v_stride_b; p.v_h = a->v_stride_h;
  p.g = a->g; p.g_b = a->g_stride_b; p.g_h = a->g_stride_h;
  p.beta = a->beta; p.beta_b = a->beta_stride_b; p.beta_h = a->beta_stride_h;
  p.idx = a->state_batch_indices;
  p.out = a->out; p.o_b = a->out_stride_b; p.o_h = a->out_stride_h;
  p.status = a->status;
  const dim3 grid(p.H * p.ns, a->batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dstate == 64)
    nssm::delta_step_kernel<64><<<grid, p.rows * 4, 0, st>>>(p);
  else
    nssm::delta_step_kernel<128><<<grid, p.rows * 4, 0, st>>>(p);
  return launched("delta_step_kernel");
}

size_t nssm_delta_scan_workspace_bytes(int32_t batch, int32_t seqlen, int32_t nheads, int32_t ngroups, int32_t dstate,
                                       int32_t packed) {
  if (batch <= 0 || seqlen <= 0 || nheads <= 0 || ngroups <= 0) return 0;
  const size_t img = dstate == 64 ? nssm::kImgBytes<64> : nssm::kImgBytes<128>;
  return (size_t)ws_chunks(batch, seqlen, packed) * (ngroups * img + (size_t)nheads * nssm::kBlkBytes);
}

int nssm_delta_scan(const nssm_delta_scan_args* a, void* stream) {
  if (!a) return fail(NSSM_ERR_INVALID, "args is NULL");
  if (a->batch < 0 || a->batch > 65535) return fail(NSSM_ERR_INVALID, "batch %d outside [0, 65535]", a->batch);
  if (a->seqlen < 0 || a->seqlen > (1 << 30)) return fail(NSSM_ERR_INVALID, "seqlen %d out of range", a->seqlen);
  int rc = check_dims(a->nheads, a->ngroups, a->headdim, a->dstate);
  if (rc) return rc;
  if (!io_ok(a->g_dtype) || !io_ok(a->beta_dtype)) return fail(NSSM_ERR_INVALID, "g / beta dtype must be F32 or BF16");
  if (a->batch == 0) return NSSM_OK;
  const bool tok = a->seqlen > 0;   // without tokens only the states move
  if (tok && (!a->q || !a->k || !a->v || !a->g || !a->beta || !a->y))
    return fail(NSSM_ERR_INVALID, "q/k/v/g/beta/y must be non-NULL");
  if (tok && (!al(a->q, 16) || !al(a->k, 16) || !al(a->v, 16) || !al(a->y, 16)))
    return fail(NSSM_ERR_INVALID, "q / k / v / y must be 16-byte aligned");
  if ((a->q_stride_b | a->q_stride_t | a->k_stride_b | a->k_stride_t | a->v_stride_b | a->v_stride_t | a->y_stride_b |
       a->y_stride_t) & 7)
    return fail(NSSM_ERR_INVALID, "q / k / v / y strides must be multiples of 8 elements");
  if (!al(a->initial_states, 16) || !al(a->final_states, 16) || ((a->init_stride_b | a->final_stride_b) & 3))
    return fail(NSSM_ERR_INVALID, "states must be 16-byte aligned");
  const int64_t row = (int64_t)a->nheads * a->headdim * a->dstate;
  if (a->final_states && a->batch > 1 && a->final_stride_b < row)
    return fail(NSSM_ERR_INVALID, "final_stride_b smaller than a state");
  const int64_t yrow = (int64_t)a->nheads * a->headdim;
  if ((a->seqlen > 1 && llabs(a->y_stride_t) < yrow) ||
      (!a->cu_seqlens && tok && a->batch > 1 && llabs(a->y_stride_b) < yrow))
    return fail(NSSM_ERR_INVALID, "tokens of y share memory");
  if (ws_chunks(a->batch, a->seqlen, a->cu_seqlens != nullptr) > (1 << 30)) return fail(NSSM_ERR_INVALID, "batch * seqlen too large");
  nssm::DeltaScanParams p{};
  p.B = a->batch; p.T = a->seqlen; p.H = a->nheads; p.G = a->ngroups; p.P = a->headdim;
  p.g_bf16 = a->g_dtype == NSSM_BF16; p.beta_bf16 = a->beta_dtype == NSSM_BF16;
  p.scale = a->scale;
  p.q = static_cast<const __nv_bfloat16*>(a->q); p.q_b = a->q_stride_b; p.q_t = a->q_stride_t;
  p.k = static_cast<const __nv_bfloat16*>(a->k); p.k_b = a->k_stride_b; p.k_t = a->k_stride_t;
  p.v = static_cast<const __nv_bfloat16*>(a->v); p.v_b = a->v_stride_b; p.v_t = a->v_stride_t;
  p.g = a->g; p.g_b = a->g_stride_b; p.g_t = a->g_stride_t;
  p.beta = a->beta; p.beta_b = a->beta_stride_b; p.beta_t = a->beta_stride_t;
  p.cu = a->cu_seqlens;
  p.init = a->initial_states; p.init_b = a->init_stride_b;
  p.y = static_cast<__nv_bfloat16*>(a->y); p.y_b = a->y_stride_b; p.y_t = a->y_stride_t;
  p.fin = a->final_states; p.fin_b = a->final_stride_b;
  p.status = a->status;
  p.polls = nssm_host::wait_polls();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = nssm_delta_scan_workspace_bytes(a->batch, a->seqlen, a->nheads, a->ngroups, a->dstate,
                                                    a->cu_seqlens != nullptr);
  if (need && (!a->workspace || !al(a->workspace, 32) || a->workspace_bytes < need))
    return fail(NSSM_ERR_INVALID, "a 32-byte aligned workspace of %zu bytes is needed (got %zu)", need, a->workspace_bytes);
  nssm::DeltaChunkParams c{};
  c.s = p;
  c.stuck = nssm_host::inject_stuck();
  c.chunks = (int)ws_chunks(a->batch, a->seqlen, a->cu_seqlens != nullptr);
  c.per_seq = (a->seqlen + kC - 1) / kC;
  c.tiles = a->headdim / 16;
  c.tile_groups = (a->nheads / a->ngroups * c.tiles + nssm::kWarps - 1) / nssm::kWarps;
  // four tiles from a multiple of four on lie in one or two heads of two tiles or more
  c.heads = c.tiles == 1 ? nssm::kWarps : c.tiles % nssm::kWarps ? 2 : 1;
  return a->dstate == 64 ? launch_chunks<64>(c, a->workspace, st) : launch_chunks<128>(c, a->workspace, st);
}

}  // extern "C"
