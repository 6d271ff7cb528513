// Internal declarations of the paged cache's translation units.
#pragma once

#include <algorithm>

#include "../../include/ar_pages.h"
#include "ar_hip_internal.h"
#include "page_index.h"

inline size_t page_elem_bytes(int dtype) { return dtype == AR_DTYPE_F32 ? 4 : 2; }
inline int page_shift_of(const ar_pages* p) { return __builtin_ctz((unsigned)p->page_rows); }

// Argument checks; `what` names the call in the messages.
int page_check(const ar_pages* p, bool table, const char* what);
int page_check_chunks(const ar_pages* p, const ar_chunks* c, const char* what);
// Extents under AR_HIP_CHECK_PTRS.
int page_check_ranges(const ar_pages* p, const char* what);
int page_check_chunk_ranges(const ar_chunks* c, const char* what);
