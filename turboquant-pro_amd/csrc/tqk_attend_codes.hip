// Launches of the attention of few queries over the codes of an fp16 cache
// (tqk_attend_codes_kernels.h), for tqk_attend.
#include "tqk_attend_codes_kernels.h"

namespace {

template <int D, int VB, bool TILED>
void launch_keys(const FewArgs& a, dim3 grid, hipStream_t st) {
  if (a.d.key_grid == 2)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, VB, true, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else if (a.d.key_bits == 4)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 4, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else if (a.d.key_bits == 3)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 3, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 2, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
}
template <int D, bool TILED>
void launch_values(const FewArgs& a, dim3 grid, hipStream_t st) {
  if (a.d.value_bits == 2)
    launch_keys<D, 2, TILED>(a, grid, st);
  else if (a.d.value_bits == 3)
    launch_keys<D, 3, TILED>(a, grid, st);
  else
    launch_keys<D, 4, TILED>(a, grid, st);
}
template <int D>
void launch_few(const FewArgs& a, dim3 grid, hipStream_t st) {
  if constexpr (D == TQK_D) {
    if (v_tiled(a.d.group_tokens, a.d.page_tokens, D, 0))
      launch_values<D, true>(a, grid, st);
    else
      launch_values<D, false>(a, grid, st);
  } else {
    launch_values<D, false>(a, grid, st);
  }
  if (a.n_splits > 1)
    hipLaunchKernelGGL(tqk_attend_join<D>, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace

size_t tqk_few_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t) { return few_plan(d, t).ws_bytes; }

int tqk_run_few(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace, size_t workspace_bytes,
                void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const FewPlan fp = few_plan(d, t);
  if (workspace_bytes < fp.ws_bytes) return TQK_EWORKSPACE;
  if (fp.groups > (1LL << 22)) return TQK_EINVAL;  // (512 threads each: fewer than 2^32)
  FewArgs a{};
  a.d = *d;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.out = out;
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + (size_t)fp.n_splits * fp.rows * d->head_dim;
  a.rows = fp.rows;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = t->q_stride[i];
    a.o_stride[i] = t->o_stride[i];
  }
  a.q_len = t->q_len;
  a.max_len = t->max_len;
  a.window = t->window;
  a.sinks = t->sinks;
  a.out_type = t->out_type;
  a.per_item = fp.per_item;
  a.q_items = fp.q_items;
  a.n_splits = fp.n_splits;
  const dim3 grid((unsigned)fp.groups);
  if (d->head_dim == 64)
    launch_few<64>(a, grid, st);
  else if (d->head_dim == 128)
    launch_few<128>(a, grid, st);
  else
    launch_few<256>(a, grid, st);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}
