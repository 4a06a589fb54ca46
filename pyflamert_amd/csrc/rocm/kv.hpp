// The paged key/value cache handle.
#pragma once

#include "common.hpp"
#include "kv_index.hpp"

// The caller's pools: element d of head h of the token in slot s is at
// (s / page_size) * page_stride + h * head_stride + (s % page_size) * token_stride + d.
struct pfr_kv {
    void* k = nullptr;
    void* v = nullptr;
    pfr_dtype dtype = PFR_F32;
    int64_t pages = 0, page_size = 0, heads = 0, dim = 0;
    int64_t page_stride = 0, head_stride = 0, token_stride = 0;
};
