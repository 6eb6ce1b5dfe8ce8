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

// The kept tokens of a sequence, at places path[0], path[1], .. of its n new ones, go to
// the places 0, 1, ..: row length - n + path[j] of the cache to row length - n + j. A
// place that is not in j .. n - 1 is no move. As no row is read behind its own write
// (path[j] >= j, and rows below j are written before) a thread that takes the same 16
// bytes of all rows, in order, needs no other one's. Bound by launch and by four loads
// after one another (offsets, path, page table, rows); the rows of eight moves are in
// flight at once. 32 layers of one sequence 3.8 us; 64 sequences of 40 heads, 4 layers 12 us,
// 4.1 TB/s.
__global__ __launch_bounds__(256) void keep_kernel(KeepCall c) {
    struct Move {
        int32_t from_page, from_at, to_page, to_at;
    };
    __shared__ Move moves[256];
    __shared__ int count_of[4];
    const int b = blockIdx.y, layer = blockIdx.z >> 1, tid = threadIdx.x;
    const bool is_v = blockIdx.z & 1;
    const int off = min(max(c.offsets[b], 0), c.tokens), n = min(max(c.offsets[b + 1], 0), c.tokens) - off;
    const int count = min(c.counts[b], n);
    const int64_t first = int64_t(c.lengths[b]) - n;
    const Rows rows = is_v ? c.v_rows : c.k_rows;
    const int shift = c.dim == 128 ? 4 : 3, piece = blockIdx.x * 256 + tid;
    const bool active = piece < c.kv_heads << shift;
    uint16_t* base = static_cast<uint16_t*>(is_v ? c.v_cache : c.k_cache) + layer * (is_v ? c.v_layer : c.k_layer) +
                     (piece >> shift) * rows.head + (piece & ((1 << shift) - 1)) * 8;
    auto entry = [&](int64_t position, int& at) {
        if (position < 0 || position >= int64_t(c.table_width) * c.page.d) return -1;
        const uint32_t p = static_cast<uint32_t>(position), q = __umulhi(p, c.page.m), rest = p - q * c.page.d;
        const bool more = rest >= c.page.d;
        at = static_cast<int>(more ? rest - c.page.d : rest);
        const int page = c.table[int64_t(b) * c.table_width + q + (more ? 1 : 0)];
        return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.pages) ? page : -1;
    };
    for (int from = 0; from < count; from += 256) {
        // Thread j looks up move j; the moves that there are move up.
        const int j = from + tid, place = j < count ? c.path[off + j] : -1;
        Move m{-1, 0, -1, 0};
        if (place > j && place < n) {
            m.from_page = entry(first + place, m.from_at);
            m.to_page = entry(first + j, m.to_at);
        }
        const bool there = m.from_page >= 0 && m.to_page >= 0;
        const uint64_t all = __ballot(there);
        __syncthreads();
        if ((tid & 63) == 0) count_of[tid >> 6] = __popcll(all);
        __syncthreads();
        int at = __popcll(all & ((uint64_t(1) << (tid & 63)) - 1)), total = 0;
        for (int w = 0; w < 4; ++w) {
            at += w < tid >> 6 ? count_of[w] : 0;
            total += count_of[w];
        }
        if (there) moves[at] = m;
        __syncthreads();
        if (!active) continue;
        constexpr int kAhead = 8;
        for (int i = 0; i < total; i += kAhead) {
            u32x4 x[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                const Move& move = moves[min(i + e, total - 1)];
                x[e] = *reinterpret_cast<const u32x4*>(base + move.from_page * rows.batch + move.from_at * rows.token);
            }
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                if (i + e >= total) break;
                const Move& move = moves[i + e];
                *reinterpret_cast<u32x4*>(base + move.to_page * rows.batch + move.to_at * rows.token) = x[e];
            }
        }
    }
}

// Pages to pages. Bound by memory, or for few pages by launch: 1.05 GB in 408 us, reading and
// writing 5.1 TB/s; a page of 32 layers 3.9 us.
constexpr int kPieces = 4;  // of 16 bytes that a thread takes
__global__ __launch_bounds__(256) void copy_kernel(CopyCall c) {
    const int layer = blockIdx.z >> 1;
    const bool is_v = blockIdx.z & 1;
    const int from = c.moves[blockIdx.y][0], to = c.moves[blockIdx.y][1];
    const int64_t page = is_v ? c.v_page : c.k_page, outer = is_v ? c.v_outer : c.k_outer, inner = is_v ? c.v_inner : c.k_inner;
    uint16_t* base = static_cast<uint16_t*>(is_v ? c.v_cache : c.k_cache) + layer * (is_v ? c.v_layer : c.k_layer);
    const uint16_t* src = base + from * page;
    uint16_t* dst = base + to * page;
    const int shift = c.dim == 128 ? 4 : 3;
    int64_t at[kPieces];
    u32x4 x[kPieces];
#pragma unroll
    for (int e = 0; e < kPieces; ++e) {
        const uint32_t piece = min((blockIdx.x * kPieces + e) * 256 + threadIdx.x, c.pieces - 1), row = piece >> shift;
        const uint32_t near = __umulhi(row, c.inner.m), rest = row - near * c.inner.d;
        const bool more = rest >= c.inner.d;
        at[e] = (near + (more ? 1 : 0)) * outer + (more ? rest - c.inner.d : rest) * inner + (piece & ((1u << shift) - 1)) * 8;
        x[e] = *reinterpret_cast<const u32x4*>(src + at[e]);
    }
#pragma unroll
    for (int e = 0; e < kPieces; ++e) *reinterpret_cast<u32x4*>(dst + at[e]) = x[e];
}
}  // namespace

int launch_keep(const KeepCall& c, hipStream_t stream) {
    const int64_t pieces = int64_t(c.kv_heads) * c.dim / 8;
    const dim3 grid(static_cast<unsigned>((pieces + 255) / 256), static_cast<unsigned>(c.batch), static_cast<unsigned>(c.layers * 2));
    hipLaunchKernelGGL(keep_kernel, grid, dim3(256), 0, stream, c);
    return check_launch("keep_kernel");
}

int launch_copy(const CopyCall& c, hipStream_t stream) {
    constexpr int64_t kGroup = 256 * kPieces;
    const dim3 grid(static_cast<unsigned>((c.pieces + kGroup - 1) / kGroup), static_cast<unsigned>(c.count), static_cast<unsigned>(c.layers * 2));
    hipLaunchKernelGGL(copy_kernel, grid, dim3(256), 0, stream, c);
    return check_launch("copy_kernel");
}

int launch_append(const AppendCall& c, hipStream_t stream) {
    hipLaunchKernelGGL(append_kernel, dim3(static_cast<unsigned>((c.tokens + 3) / 4)), dim3(256), 0, stream, c);
    return check_launch("append_kernel");
}

}  // namespace ab
