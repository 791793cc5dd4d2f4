// Fused decode-step attention over the two-tier TurboQuant KV cache (gfx950):
// launches and C ABI of the kernels in tqk_decode_kernels.h.
#include "tqk_decode_kernels.h"

namespace {

template <int GQ, int KB>
void launch_mfma_kb(const DecodeArgs& a, dim3 g1, hipStream_t st) {
  if (a.d.key_grid == 2)  // PolarQuant keys: value_bits == key_bits
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, KB, KB, true>), g1, dim3(kMThreads), 0, st, a);
  else if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 2, KB, false>), g1, dim3(kMThreads), 0, st, a);
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 3, KB, false>), g1, dim3(kMThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 4, KB, false>), g1, dim3(kMThreads), 0, st, a);
}

template <int GQ, int D>
void launch_valu(const DecodeArgs& a, dim3 grid, hipStream_t st) {
  if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 2, D, false>), grid, dim3(kThreads), 0, st, SplitArgs<false>{a});
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 3, D, false>), grid, dim3(kThreads), 0, st, SplitArgs<false>{a});
  else
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 4, D, false>), grid, dim3(kThreads), 0, st, SplitArgs<false>{a});
}

template <int GQ>
hipError_t launch_split(const DecodeArgs& a, dim3 grid, hipStream_t st) {
  if (!mfma_path(a.d)) {
    if (a.d.head_dim == 64)
      launch_valu<GQ, 64>(a, grid, st);
    else if (a.d.head_dim == 128)
      launch_valu<GQ, 128>(a, grid, st);
    else
      launch_valu<GQ, 256>(a, grid, st);
    return hipGetLastError();
  }
  // one-dimensional over (split, kv head, seq) items
  const dim3 g1(grid.x * grid.y * grid.z);
  if (a.d.key_bits == 4)
    launch_mfma_kb<GQ, 4>(a, g1, st);
  else if (a.d.key_bits == 3)
    launch_mfma_kb<GQ, 3>(a, g1, st);
  else
    launch_mfma_kb<GQ, 2>(a, g1, st);
  return hipGetLastError();
}

DecodeArgs make_args(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const Plan& pl, int batch,
                     const void* q, const int32_t* seq_lens, const WsView& w) {
  const int ns = pl.n_cold_splits + pl.n_hot_splits;
  const size_t per = (size_t)batch * d->n_q_heads * ns;
  DecodeArgs a;
  a.d = *d;
  a.p = *p;
  a.q = q;
  a.seq_lens = seq_lens;
  a.arrive = w.arrive;
  a.pm = reinterpret_cast<float*>(w.partials);
  a.pl = a.pm + per;
  a.pacc = a.pl + per;
  a.n_cold_splits = pl.n_cold_splits;
  a.n_hot_splits = pl.n_hot_splits;
  a.groups_per_split = pl.groups_per_split;
  a.wave_blocks = pl.wave_blocks;
  a.hot_per_split = pl.hot_per_split;
  a.split_base = 0;
  a.batch = batch;
  a.reorder = mfma_path(*d) && (long)pl.n_cold_splits * d->n_kv_heads * batch > device_cus();
  a.out = nullptr;
  return a;
}

WsView caller_ws(const Plan& pl, void* ws) {
  return WsView{reinterpret_cast<uint32_t*>(ws), static_cast<char*>(ws) + pl.counter_bytes};
}

// Arguments every decode entry point validates the same way.
int check_decode_args(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int batch, int max_len) {
  int rc = tqk_check_desc(d);
  if (rc != TQK_OK) return rc;
  if (!p || batch <= 0 || max_len <= 0) return TQK_EINVAL;
  if (d->key_grid == 2 && !p->knorm) return TQK_EINVAL;
  if (batch > counter_seqs(*d)) return TQK_EINVAL;
  return TQK_OK;
}

// The split kernel (validated arguments); `out` non-null selects the MFMA
// kernel's in-kernel merge.
int launch_splits(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const Plan& pl, int batch,
                  const void* q, const int32_t* seq_lens, const WsView& w, void* stream,
                  float* out) {
  DecodeArgs a = make_args(d, p, pl, batch, q, seq_lens, w);
  if (out && mfma_path(*d)) a.out = out;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // (the MFMA kernel's workgroups are the coded splits; each also covers a
  // share of the hot window)
  const dim3 grid(mfma_path(*d) ? pl.n_cold_splits : pl.n_cold_splits + pl.n_hot_splits,
                  d->n_kv_heads, batch);
  hipError_t e;
  // kernels exist for 1, 2, 4 and 8 query heads per kv head; other counts
  // run on the next larger one with zero-query padding heads
  switch (d->n_q_heads / d->n_kv_heads) {
    case 1: e = launch_split<1>(a, grid, st); break;
    case 2: e = launch_split<2>(a, grid, st); break;
    case 3: case 4: e = launch_split<4>(a, grid, st); break;
    case 5: case 6: case 7: case 8: e = launch_split<8>(a, grid, st); break;
    default: return TQK_EUNSUPPORTED;
  }
  return e == hipSuccess ? TQK_OK : TQK_EHIP;
}

// tqk_merge over the partials the split kernel left (validated arguments).
int launch_merge(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const Plan& pl, int batch,
                 const WsView& w, float* out, float* m_out, float* l_out, float* acc_out,
                 void* stream) {
  const DecodeArgs a = make_args(d, p, pl, batch, nullptr, nullptr, w);
  MergeArgs m;
  m.pm = a.pm;
  m.pl = a.pl;
  m.pacc = a.pacc;
  m.pi = p->pi;
  m.n_cold_splits = pl.n_cold_splits;
  m.n_splits = pl.n_cold_splits + pl.n_hot_splits;
  m.n_q_heads = d->n_q_heads;
  m.n_kv_heads = d->n_kv_heads;
  m.out = out;
  m.m_out = m_out;
  m.l_out = l_out;
  m.acc_out = acc_out;
  const dim3 grid(d->n_kv_heads, batch);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (d->head_dim == 64)
    hipLaunchKernelGGL((tqk_merge<64, false>), grid, dim3(128), 0, st, JoinArgs<false>{m});
  else if (d->head_dim == 128)
    hipLaunchKernelGGL((tqk_merge<128, false>), grid, dim3(256), 0, st, JoinArgs<false>{m});
  else
    hipLaunchKernelGGL((tqk_merge<256, false>), grid, dim3(512), 0, st, JoinArgs<false>{m});
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}

int run_splits(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int batch, const void* q,
               const int32_t* seq_lens, int max_len, void* ws, size_t ws_bytes, void* stream,
               float* out = nullptr) {
  int rc = check_decode_args(d, p, batch, max_len);
  if (rc != TQK_OK) return rc;
  if (!q || !seq_lens) return TQK_EINVAL;
  const Plan pl = make_plan(d, batch, max_len);
  if (!ws || ws_bytes < pl.ws_bytes) return TQK_EWORKSPACE;
  return launch_splits(d, p, pl, batch, q, seq_lens, caller_ws(pl, ws), stream, out);
}

int run_merge(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int batch, int max_len, float* out,
              float* m_out, float* l_out, float* acc_out, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_decode_args(d, p, batch, max_len);
  if (rc != TQK_OK) return rc;
  if (!out && !(m_out && l_out && acc_out)) return TQK_EINVAL;
  const Plan pl = make_plan(d, batch, max_len);
  if (!ws || ws_bytes < pl.ws_bytes) return TQK_EWORKSPACE;
  return launch_merge(d, p, pl, batch, caller_ws(pl, ws), out, m_out, l_out, acc_out, stream);
}

// ---- the no-allocation decode's scratch ------------------------------------
// One zero-fill kernel for the scratch array's counter region (a kernel, not
// hipMemsetAsync, so that no memset node is recorded if a caller captures it).
__global__ void tqk_zero_words(uint32_t* p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 0u;
}

}  // namespace

// Device scratch of tqk_decode_noalloc, one copy per GPU for the life of the
// process: kNoAllocCounters arrival counters, then the split partials.  The
// array's name is a host-side stand-in: host code only ever uses the address
// hipGetSymbolAddress returns for the current device (noalloc_scratch()).
constexpr int kNoAllocCounters = 1 << 16;         // (sequence, kv head) pairs per call
constexpr size_t kNoAllocBytes = (size_t)32 << 20;  // 32 MiB per GPU
static __device__ __align__(256) uint8_t scratch[kNoAllocBytes];

namespace {

std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices];

// The current device's scratch address, resolved (and its counters zeroed,
// on `stream`) at the first call on that device.
int noalloc_scratch(hipStream_t stream, void** out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return TQK_EHIP;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess || !ptr) return TQK_EHIP;
    hipLaunchKernelGGL(tqk_zero_words, dim3(kNoAllocCounters / 256), dim3(256), 0, stream,
                       static_cast<uint32_t*>(ptr), kNoAllocCounters);
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
    g_scratch_ptr[dev] = ptr;
  }
  *out = g_scratch_ptr[dev];
  return TQK_OK;
}

}  // namespace

extern "C" {

int tqk_version(void) { return 9; }

int tqk_check_desc(const tqk_cache_desc* d) {
  if (!d) return TQK_EINVAL;
  if (!head_dim_ok(d->head_dim)) return TQK_EUNSUPPORTED;
  if (d->input_f32 != 0 && d->input_f32 != 1) return TQK_EINVAL;
  if (d->key_bits < 2 || d->key_bits > 4) return TQK_EUNSUPPORTED;
  if (d->key_grid < 0 || d->key_grid > 2) return TQK_EINVAL;
  // NF4 is a 4-bit grid; 3- and 2-bit keys are uniform or PolarQuant
  if (d->key_bits != 4 && d->key_grid == 0) return TQK_EUNSUPPORTED;
  // PolarQuant keys share the value codebook and carry no side-list
  if (d->key_grid == 2 && (d->key_bits != d->value_bits || d->outliers_per_channel != 0)) return TQK_EUNSUPPORTED;
  if (d->value_bits < 2 || d->value_bits > 4) return TQK_EUNSUPPORTED;
  if (d->zero_point < 0 || d->zero_point > 2 || (d->zero_point != 0 && d->key_grid != 0))
    return TQK_EINVAL;
  if (d->n_kv_heads <= 0 || d->n_q_heads <= 0 || d->n_q_heads % d->n_kv_heads) return TQK_EINVAL;
  const int gq = d->n_q_heads / d->n_kv_heads;
  if (gq < 1 || gq > 8) return TQK_EUNSUPPORTED;
  if (d->hot_window < 1) return TQK_EINVAL;
  if (d->group_tokens != (d->hot_window + 1) / 2) return TQK_EINVAL;
  if (d->group_tokens < 1 || d->group_tokens > TQK_MAX_G) return TQK_EUNSUPPORTED;
  if (d->page_tokens < 1 || d->group_tokens % d->page_tokens) return TQK_EINVAL;
  if (d->hot_ring < d->hot_window) return TQK_EINVAL;
  if (d->outliers_per_channel < 0 || d->outlier_cap < 0) return TQK_EINVAL;
  if (d->max_groups_per_seq < 0 || d->max_pages_per_seq < 0 || d->n_pages < 1) return TQK_EINVAL;
  return TQK_OK;
}

size_t tqk_decode_workspace_bytes(const tqk_cache_desc* d, int32_t batch, int32_t max_len) {
  if (!d || batch <= 0 || max_len <= 0 || batch > counter_seqs(*d)) return 0;
  return make_plan(d, batch, max_len).ws_bytes;
}

int tqk_decode(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch,
               const void* q, const int32_t* seq_lens, int32_t max_len, float* out,
               void* workspace, size_t workspace_bytes, void* stream) {
  if (!out) return TQK_EINVAL;
  int rc = run_splits(d, p, batch, q, seq_lens, max_len, workspace, workspace_bytes, stream, out);
  if (rc != TQK_OK) return rc;
  // the MFMA kernel merged in its last workgroups
  if (mfma_path(*d)) return TQK_OK;
  return run_merge(d, p, batch, max_len, out, nullptr, nullptr, nullptr, workspace,
                   workspace_bytes, stream);
}

int tqk_decode_noalloc(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch,
                       const void* q, const int32_t* seq_lens, int32_t max_len, float* out,
                       void* stream) {
  int rc = check_decode_args(d, p, batch, max_len);
  if (rc != TQK_OK) return rc;
  if (!q || !seq_lens || !out) return TQK_EINVAL;
  const Plan pl = make_plan(d, batch, max_len);
  constexpr size_t kCounterBytes = (size_t)kNoAllocCounters * sizeof(uint32_t);
  if ((size_t)batch * d->n_kv_heads > (size_t)kNoAllocCounters ||
      pl.partial_bytes > kNoAllocBytes - kCounterBytes)
    return TQK_EWORKSPACE;
  void* base = nullptr;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  rc = noalloc_scratch(st, &base);
  if (rc != TQK_OK) return rc;
  const WsView w{static_cast<uint32_t*>(base), static_cast<char*>(base) + kCounterBytes};
  rc = launch_splits(d, p, pl, batch, q, seq_lens, w, stream, out);
  if (rc != TQK_OK || mfma_path(*d)) return rc;
  return launch_merge(d, p, pl, batch, w, out, nullptr, nullptr, nullptr, stream);
}

int tqk_decode_partials(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch,
                        const void* q, const int32_t* seq_lens, int32_t max_len,
                        float* m, float* l, float* acc, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (!m || !l || !acc) return TQK_EINVAL;
  int rc = run_splits(d, p, batch, q, seq_lens, max_len, workspace, workspace_bytes, stream);
  if (rc != TQK_OK) return rc;
  return run_merge(d, p, batch, max_len, nullptr, m, l, acc, workspace, workspace_bytes, stream);
}

int tqk_decode_splits(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch,
                      const void* q, const int32_t* seq_lens, int32_t max_len,
                      void* workspace, size_t workspace_bytes, void* stream) {
  return run_splits(d, p, batch, q, seq_lens, max_len, workspace, workspace_bytes, stream);
}

int tqk_decode_merge(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch,
                     int32_t max_len, float* out, void* workspace, size_t workspace_bytes,
                     void* stream) {
  if (!out) return TQK_EINVAL;
  return run_merge(d, p, batch, max_len, out, nullptr, nullptr, nullptr, workspace,
                   workspace_bytes, stream);
}

}  // extern "C"
