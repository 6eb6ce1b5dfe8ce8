// New keys and values into a paged cache: row i of sequence b (of its n new
// tokens) goes to position length_b - n + i, page table[b][position / page].
// One wave per row, whose place is the same for all its heads; a copy, bound by
// memory (9,360 rows of 40 heads 76 us, 5.0 TB/s) or, for single tokens, by the three
// loads that find the place (32 rows of 8 heads 3.2 us).
#include "cache.hpp"

namespace ab {
namespace {

__global__ __launch_bounds__(256) void append_kernel(AppendCall c) {
    touch(c.k, c.v, c.k_cache_rows.token, c.v_cache_rows.token, c.table, c.batch);
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= c.tokens) return;
    // The sequence: the last one that starts at or before the row.
    int before = 0;
    for (int at = 0; at < c.batch; at += 64) {
        const int b = min(at + lane, c.batch - 1);
        before += __popcll(__ballot(at + lane < c.batch && c.offsets[b] <= row));
    }
    const int b = __builtin_amdgcn_readfirstlane(before) - 1;
    if (b < 0) return;
    const int next = min(c.offsets[b + 1], c.tokens);  // as the attention bounds it, so that both see the same positions
    if (row >= next) return;
    const int64_t position = int64_t(c.lengths[b]) - next + row;
    if (position < 0 || position >= int64_t(c.table_width) * c.page.d) return;
    uint32_t in_page;
    const uint32_t index = c.page.quotient(static_cast<uint32_t>(position), in_page);
    const int entry = c.table[int64_t(b) * c.table_width + index];
    if (static_cast<uint32_t>(entry) >= static_cast<uint32_t>(c.pages)) return;

    const int chunks = c.dim / 8, work = c.kv_heads * chunks;  // 16-byte pieces
    const uint16_t* src[2] = {static_cast<const uint16_t*>(c.k) + int64_t(row) * c.k_rows.token,
                              static_cast<const uint16_t*>(c.v) + int64_t(row) * c.v_rows.token};
    uint16_t* dst[2] = {static_cast<uint16_t*>(c.k_cache) + entry * c.k_cache_rows.batch + in_page * c.k_cache_rows.token,
                        static_cast<uint16_t*>(c.v_cache) + entry * c.v_cache_rows.batch + in_page * c.v_cache_rows.token};
    const int shift = c.dim == 128 ? 4 : 3;
#pragma unroll 2
    for (int i = lane; i < work; i += 64) {
        const int head = i >> shift, at = (i & (chunks - 1)) * 8;
        const u32x4 a = *reinterpret_cast<const u32x4*>(src[0] + head * c.k_rows.head + at);
        const u32x4 d = *reinterpret_cast<const u32x4*>(src[1] + head * c.v_rows.head + at);
        *reinterpret_cast<u32x4*>(dst[0] + head * c.k_cache_rows.head + at) = a;
        *reinterpret_cast<u32x4*>(dst[1] + head * c.v_cache_rows.head + at) = d;
    }
}
}  // namespace

int launch_append(const AppendCall& c, hipStream_t stream) {
    hipLaunchKernelGGL(append_kernel, dim3(static_cast<unsigned>((c.tokens + 3) / 4)), dim3(256), 0, stream, c);
    return check_launch("append_kernel");
}

}  // namespace ab
