// Attention of few queries over the codes of an fp16 cache (tqk_attend_codes.hip),
// for tqk_attend; arguments checked by the caller.
#pragma once

#include "tqk_common.h"

size_t tqk_few_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t);
int tqk_run_few(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace, size_t workspace_bytes, void* stream);
