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

int launch_append(const AppendCall& call, hipStream_t stream);

}  // namespace ab
