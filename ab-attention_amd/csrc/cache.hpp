// One call of the append kernel.
#pragma once

#include "window.hpp"

namespace ab {

struct AppendCall {
    const void *k, *v;
    void *k_cache, *v_cache;
    Rows k_rows, v_rows;              // batch unused
    Rows k_cache_rows, v_cache_rows;  // batch: from a page to the next
    const int32_t *table, *lengths, *offsets;
    int32_t batch, kv_heads, dim, tokens, table_width, pages;
    Divisor page;
};

// Kept tokens to the first places of their sequences' new ones, in `layers` caches.
struct KeepCall {
    void *k_cache, *v_cache;
    Rows k_rows, v_rows;  // batch: from a page to the next
    int64_t k_layer, v_layer;
    const int32_t *table, *lengths, *offsets, *path, *counts;
    int32_t layers, batch, kv_heads, dim, tokens, table_width, pages;
    Divisor page;
};

constexpr int kMovesAtOnce = 256;

// Pages to pages, in `layers` caches. Rows of a page in the order of memory: `inner` of
// them (heads, or tokens) at the inner stride, then the next at the outer one.
struct CopyCall {
    void *k_cache, *v_cache;
    int64_t k_layer, v_layer, k_page, v_page, k_outer, v_outer, k_inner, v_inner;
    Divisor inner;
    uint32_t pieces;  // of 16 bytes in a page
    int32_t layers, dim, count;
    int32_t moves[kMovesAtOnce][2];  // from, to
};

int launch_append(const AppendCall& call, hipStream_t stream);
int launch_keep(const KeepCall& call, hipStream_t stream);
int launch_copy(const CopyCall& call, hipStream_t stream);

}  // namespace ab
