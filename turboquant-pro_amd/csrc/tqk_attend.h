// Attention of few queries over the codes of an fp16 cache (tqk_attend_codes.hip),
// for tqk_attend; arguments checked by the caller.
#pragma once

#include "tqk_common.h"

size_t tqk_few_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t);
bool tqk_few_fits(const tqk_cache_desc* d, const tqk_attend_desc* t);  // within one launch (else TQK_EINVAL)
int tqk_run_few(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace, size_t workspace_bytes, void* stream);

// The checks of tqk_attend and its kin, before any GPU work: of the descriptors, and
// whether every buffer that a cache of this form has is there.
int tqk_check_attend(const tqk_cache_desc* d, const tqk_attend_desc* t);
bool tqk_have_buffers(const tqk_cache_desc& d, const tqk_cache_ptrs& p);
