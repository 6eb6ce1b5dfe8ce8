// Windowed causal attention, forward, over strided tensors or a paged cache.
//
// For the query at position p and the keys t that its mask leaves (WindowMask),
//   z_t = q . k_t * scale * log2(e),  o = sum_t 2^(z_t - m) v_t / sum_t 2^(z_t - m),
//   lse = m + log2(sum_t 2^(z_t - m)),
// with the running maximum and sum of an online softmax in float32; a query
// that sees nothing gets o = 0 and lse = -inf.
//
// One workgroup of four waves takes 128 rows of one K/V head of one batch item:
// tokens, or over a cache (token, query head of the group) pairs, so that the
// heads that share keys read them once. It visits only tiles of 32 keys that
// some of its rows see: the sinks' tiles, then the window's.
#include <algorithm>

#include "window.hpp"

namespace ab {
namespace {

// What a workgroup works on. The same in all its lanes.
struct WindowUnit {
    int b, kv_head, head;  // head: the query head, or the first one of the group
    int tile;              // rows tile * kWindowRows .. of the batch item's packed rows
    int n;                 // its new tokens
    int off;               // their first row in the packed tensor (0 without offsets)
    int first;             // position of its first new token
    int length;            // keys of it
};

template <bool kPaged>
__device__ __forceinline__ bool window_unit(const WindowCall& c, uint32_t id, int tiles, WindowUnit& u) {
    int head;
    if constexpr (!kPaged) {
        if (!window_place(id, c.batch * c.heads, tiles, head, u.tile)) return false;
        u.b = head / c.heads;
        u.head = head - u.b * c.heads;
        u.kv_head = u.head / static_cast<int>(c.group.d);
        u.n = c.tokens;
        u.off = 0;
        u.first = 0;
        u.length = c.lengths ? min(max(c.lengths[u.b], 0), c.tokens) : c.tokens;
        return true;
    } else {
        // Sequence b's tiles take the slots from offsets[b] * group / 128 + b on:
        // never fewer than it needs, so no sum over the sequences is wanted.
        int slot;
        if (!window_place(id, c.kv_heads, tiles, head, slot)) return false;
        u.kv_head = head;
        u.head = head * c.group.d;
        const int lane = threadIdx.x & 63;
        int before = 0;
        for (int at = 0; at < c.batch; at += 64) {
            const int b = min(at + lane, c.batch - 1);
            const int64_t start = int64_t(min(max(c.offsets[b], 0), c.tokens)) * c.group.d / kWindowRows + b;
            before += __popcll(__ballot(at + lane < c.batch && start <= slot));
        }
        u.b = __builtin_amdgcn_readfirstlane(before) - 1;
        if (u.b < 0) return false;
        u.off = min(max(c.offsets[u.b], 0), c.tokens);
        u.n = min(max(c.offsets[u.b + 1], 0), c.tokens) - u.off;
        u.tile = slot - static_cast<int>(int64_t(u.off) * c.group.d / kWindowRows + u.b);
        if (int64_t(u.tile) * kWindowRows >= int64_t(u.n) * c.group.d) return false;
        u.length = static_cast<int>(min(int64_t(max(c.lengths[u.b], 0)), int64_t(c.table_width) * c.page.d));
        u.first = u.length - u.n;
        return true;
    }
}

template <class T, int D>
struct WindowTile {
    static constexpr int kSteps = D / 32;                  // MFMA k-steps of S
    static constexpr int kBlocks = D / 16;                 // 16-dim blocks of O
    static constexpr int kQuadBytes = 4 * D * 2;           // four keys of K (or V)
    static constexpr int kBytes = kWindowKeys * D * 2;     // K (or V) of one tile
    static constexpr int kOps = D / 64;                    // transfers of a wave for K (or V) of a tile
    static constexpr int kOpKeys = 1024 / (2 * D);         // keys of a transfer
};

template <class T, int D, bool kPaged, bool kSplit>
__global__ __launch_bounds__(kWindowThreads, 2) void window_kernel(WindowCall c, int tiles_per_head) {
    using Tile = WindowTile<T, D>;
    constexpr int kSteps = Tile::kSteps, kBlocks = Tile::kBlocks;
    __shared__ __align__(16) unsigned char smem[4 * Tile::kBytes];  // two stages of K, two of V

    WindowUnit u;
    if (!window_unit<kPaged>(c, blockIdx.x, tiles_per_head, u)) return;
    const int group = kPaged ? c.group.d : 1;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;

    // Bounds of the rows r0 .. r1 of the tile that exist: keys that some row
    // sees, and those that every row sees.
    const WindowMask mask = c.mask;
    const int row0 = u.tile * kWindowRows, rows = min(kWindowRows, u.n * group - row0);
    auto token_at = [&](int r) { return kPaged ? (row0 + r) / group : row0 + r; };
    const int p_first = max(u.first + token_at(0), 0), p_last = min(u.first + token_at(rows - 1), u.length - 1);
    TileRange range;
    range.set(mask, p_first, p_last, u.length);
    const int end = range.end;
    int tile0 = 0, tiles = range.tiles;
    if constexpr (kSplit) {
        const int part = blockIdx.y;
        tile0 = static_cast<int>(int64_t(tiles) * part / c.parts);
        tiles = static_cast<int>(int64_t(tiles) * (part + 1) / c.parts) - tile0;
    }

    // Q as the B operand of S^T = K Q^T: row 16j + li of the wave's 32, dims
    // 32s + 8lg .. + 7. The row's own bounds; all zero for a row without keys.
    u32x4 bq[2][kSteps];
    int low[2], seen[2], sink[2];  // keys low .. low + seen - 1 and 0 .. sink - 1
    int64_t out_at[2], stat_at[2];
    bool stored[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = wave * 32 + 16 * j + li;
        stored[j] = r < rows;
        const int packed = row0 + min(r, rows - 1);
        const int token = kPaged ? packed / group : packed, head = u.head + (kPaged ? packed - token * group : 0);
        const uint16_t* qrow = static_cast<const uint16_t*>(c.q) + u.b * c.q_rows.batch + head * c.q_rows.head +
                               int64_t(u.off + token) * c.q_rows.token + 8 * lg;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) bq[j][s] = *reinterpret_cast<const u32x4*>(qrow + 32 * s);
        const int p = u.first + token;
        const bool sees = stored[j] && p >= 0 && p < u.length;
        const int high = mask.high(max(p, 0), u.length);
        low[j] = mask.low(max(p, 0));
        seen[j] = sees ? high - low[j] : 0;
        sink[j] = sees ? min(mask.sinks, high) : 0;
        out_at[j] = u.b * c.out_rows.batch + head * c.out_rows.head + int64_t(u.off + token) * c.out_rows.token;
        stat_at[j] = u.b * c.row.batch + head * c.row.head + int64_t(u.off + token) * c.row.token;
    }
    // Tiles that every row of this wave sees need no mask: keys from full_low to
    // full_high, and those before full_sink. A wave with a row that exists but
    // sees nothing masks every tile.
    int full_low = 0, full_high = 0, full_sink = 0;
    const int wave_rows = min(32, rows - wave * 32);
    if (wave_rows > 0) {
        const int pf = u.first + token_at(wave * 32), pl = u.first + token_at(wave * 32 + wave_rows - 1);
        if (pf >= 0 && pl < u.length) {
            full_low = mask.low(pl);
            full_high = mask.high(pf, u.length);
            full_sink = min(mask.sinks, full_high);
        }
    }

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)smem));
    const char* kbase = static_cast<const char*>(c.k) + ((kPaged ? 0 : u.b * c.k_rows.batch) + u.kv_head * c.k_rows.head) * 2;
    const char* vbase = static_cast<const char*>(c.v) + ((kPaged ? 0 : u.b * c.v_rows.batch) + u.kv_head * c.v_rows.head) * 2;
    const uint32_t k_token = static_cast<uint32_t>(c.k_rows.token * 2), v_token = static_cast<uint32_t>(c.v_rows.token * 2);
    const int32_t* table = kPaged ? c.table + int64_t(u.b) * c.table_width : nullptr;

    // The page of a key (a multiple of 8): where it starts and how many of its
    // tokens exist; nothing for an entry that names no page.
    auto page_of = [&](int key, int64_t& page, uint32_t& in_page, uint32_t& there) {
        uint32_t rest;
        const uint32_t index = c.page.quotient(static_cast<uint32_t>(key), rest);
        page = 0;
        in_page = rest;
        there = 0;
        if (key < end) {
            const int entry = __builtin_amdgcn_readfirstlane(table[index]);
            if (static_cast<uint32_t>(entry) < static_cast<uint32_t>(c.pages)) {
                page = entry;
                there = min(static_cast<int>(c.page.d), end - (key - static_cast<int>(rest)));
            }
        }
    };

    // Transfers of this wave: keys 8w .. 8w + 7 of the tile, kOpKeys at a time.
    // K keeps rows of D elements whose 16-byte chunks are swizzled (position =
    // chunk ^ key); V keeps, for every four keys, blocks of 4 keys x 16 dims,
    // block m at position m ^ (quad & 1): both the row reads of K and the
    // transposing reads of V then spread over the banks.
    uint32_t k_src[Tile::kOps], v_src[Tile::kOps];
#pragma unroll
    for (int e = 0; e < Tile::kOps; ++e) {
        constexpr int kChunks = D / 8;
        const int key = lane / kChunks, pos = lane % kChunks, in_tile = 8 * wave + Tile::kOpKeys * e + key;
        k_src[e] = uint32_t(key) * k_token + uint32_t(pos ^ (in_tile % kChunks)) * 16u;
        const int quad = D == 128 ? e : lane >> 5, block = (lane >> 3) % kBlocks, r = (lane >> 1) & 3, h = lane & 1;
        v_src[e] = uint32_t((D == 128 ? 0 : 4 * quad) + r) * v_token + uint32_t(2 * (block ^ (quad & 1)) + h) * 16u;
    }
    auto transfer = [&](int t) {
        if (t >= tiles) return;
        const int key = range.key(tile0 + t) + 8 * wave;
        const uint32_t stage = (t & 1) * Tile::kBytes + wave * (8 * D * 2);
        u32x4 kbuf, vbuf;
        uint32_t at;
        if constexpr (kPaged) {
            int64_t page;
            uint32_t there;
            page_of(key, page, at, there);
            kbuf = buffer_of(kbase + page * c.k_rows.batch * 2, there ? (there - 1) * k_token + 2 * D : 0);
            vbuf = buffer_of(vbase + page * c.v_rows.batch * 2, there ? (there - 1) * v_token + 2 * D : 0);
        } else {
            at = key;
            kbuf = buffer_of(kbase, uint32_t(end - 1) * k_token + 2 * D);
            vbuf = buffer_of(vbase, uint32_t(end - 1) * v_token + 2 * D);
        }
#pragma unroll
        for (int e = 0; e < Tile::kOps; ++e) {
            buffer_to_lds(kbuf, k_src[e] + (at + Tile::kOpKeys * e) * k_token, lds0 + stage + 1024 * e);
            buffer_to_lds(vbuf, v_src[e] + (at + Tile::kOpKeys * e) * v_token, lds0 + 2 * Tile::kBytes + stage + 1024 * e);
        }
    };

    // Whether a key that some row would see lies on no page (then every tile
    // asks the table for its keys).
    bool holes = false;
    if constexpr (kPaged) {
        if (tiles > 0) {
            const int first_page = range.key(tile0) / static_cast<int>(c.page.d);
            const int last_page = (min(range.key(tile0 + tiles - 1) + kWindowKeys, end) - 1) / static_cast<int>(c.page.d);
            bool bad = false;
            for (int i = first_page + tid; i <= last_page; i += kWindowThreads)
                bad |= static_cast<uint32_t>(table[i]) >= static_cast<uint32_t>(c.pages);
            holes = __syncthreads_or(bad);
        }
    }
    auto on_page = [&](int key) {
        const uint32_t q0 = __umulhi(static_cast<uint32_t>(key), c.page.m);
        const uint32_t index = q0 + (static_cast<uint32_t>(key) - q0 * c.page.d >= c.page.d ? 1u : 0u);
        return key < end && static_cast<uint32_t>(table[min(index, static_cast<uint32_t>(c.table_width - 1))]) < static_cast<uint32_t>(c.pages);
    };

    uint32_t k_abs[kSteps], v_abs[2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) k_abs[s] = lds0 + li * (2 * D) + 16 * ((4 * s + lg) ^ (li % (D / 8)));
    {
        const int par = lg & 1, base = 2 * Tile::kBytes + lg * Tile::kQuadBytes + 32 * (li >> 2) + 8 * (li & 3);
        v_abs[0] = lds0 + base + par * 128;  // even block: position block + par
        v_abs[1] = lds0 + base - par * 128;  // odd block: position block - par
    }

    f32x4 o_acc[kBlocks][2];  // dims 16b + 4lg .. + 3 of row 16j + li
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) o_acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    transfer(0);
    for (int t = 0; t < tiles; ++t) {
        landed_and_barrier<0>();
        transfer(t + 1);
        if (wave_rows <= 0) continue;
        const int key0 = range.key(tile0 + t), stage = (t & 1) * Tile::kBytes;
        const bool masked = holes || !((key0 >= full_low && key0 + kWindowKeys <= full_high) || key0 + kWindowKeys <= full_sink);

        // S^T: keys 16h + 4lg + r of row 16j + li in sc[2h + j][r].
        f32x4 sc[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 a = lds_read16(k_abs[s] + stage + h * 16 * 2 * D);
#pragma unroll
                for (int j = 0; j < 2; ++j) sc[2 * h + j] = T::mfma16(a, bq[j][s], sc[2 * h + j]);
            }
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[x] *= c.scale_log2;
        float top[2] = {-INFINITY, -INFINITY};
        uint32_t visible[2] = {0xffu, 0xffu};  // bit 4h + r
        if (masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + 16 * h + 4 * lg;
                const bool there = !kPaged || !holes || on_page(key);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool sees = there && (static_cast<uint32_t>(key + r - low[j]) < static_cast<uint32_t>(seen[j]) ||
                                                    key + r < sink[j]);
                        if (!sees) {
                            sc[2 * h + j][r] = -INFINITY;
                            visible[j] &= ~(1u << (4 * h + r));
                        }
                    }
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[x & 1] = fmaxf(top[x & 1], sc[x][r]);
        uint32_t pw[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[j] = fmaxf(top[j], __shfl_xor(top[j], 16));
            top[j] = fmaxf(top[j], __shfl_xor(top[j], 32));
            const float m = fmaxf(m_run[j], top[j]);
            const float reference = m == -INFINITY ? 0.f : m;
            const float alpha = fast_exp2(m_run[j] - reference);
            m_run[j] = m;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float p0 = fast_exp2(sc[2 * h + j][r] - reference), p1 = fast_exp2(sc[2 * h + j][r + 1] - reference);
                    sum += p0 + p1;
                    pw[j][2 * h + r / 2] = T::pack(p0, p1);
                }
            l_run[j] = l_run[j] * alpha + sum;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) o_acc[b][j][r] *= alpha;
        }
        // O^T += V^T P^T: the MFMA's k index 8lg + 4h + r is key 16h + 4lg + r
        // on both operands, so P stays where the first product left it.
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint32_t at = v_abs[b & 1] + stage + b * 128;
            u32x4 a = __builtin_bit_cast(u32x4, __builtin_shufflevector(lds_read_transposed(at),
                                                                         lds_read_transposed(at + 4 * Tile::kQuadBytes), 0, 1, 2, 3, 4, 5, 6, 7));
            if (masked) {
                // 0 times an infinity or a NaN is no zero: values that are not finite
                // reach only the rows that see them.
                uint32_t odd = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (a[w] & T::kExponent) + T::kOverflow;
                if (__any((odd & 0x80008000u) != 0)) {
                    u32x4 finite = a, up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t bits = (a[w] >> (16 * half)) & 0xffffu, exponent = T::kExponent & 0xffffu;
                            if ((bits & exponent) != exponent) continue;
                            const bool nan = (bits & 0x7fffu) != exponent;
                            finite[w] &= half ? 0xffffu : 0xffff0000u;
                            if (nan || !(bits & 0x8000u)) up[w] |= T::kOne << (16 * half);
                            if (nan || (bits & 0x8000u)) down[w] |= T::kOne << (16 * half);
                        }
                    a = finite;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        u32x4 sees;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            sees[w] = ((visible[j] >> (2 * w)) & 1 ? T::kOne : 0u) | ((visible[j] >> (2 * w + 1)) & 1 ? T::kOne << 16 : 0u);
                        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                        const f32x4 ups = T::mfma16(up, sees, zero), downs = T::mfma16(down, sees, zero);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (ups[r] > 0.f) o_acc[b][j][r] += INFINITY;
                            if (downs[r] > 0.f) o_acc[b][j][r] -= INFINITY;
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x4 p = {pw[j][0], pw[j][1], pw[j][2], pw[j][3]};
                o_acc[b][j] = T::mfma16(a, p, o_acc[b][j]);
            }
        }
    }

#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float l = l_run[j];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (!stored[j]) continue;
        if constexpr (kSplit) {
            const int64_t at = blockIdx.y * c.rows + stat_at[j];
            if (lg == 0) c.partial_stat[at] = float2{m_run[j], l};
            if (l == 0.f) continue;
            float* dst = c.partial_o + at * D + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4*>(dst + 16 * b) = o_acc[b][j];
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            uint16_t* orow = static_cast<uint16_t*>(c.out) + out_at[j] + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const u32x2 w = {T::pack(o_acc[b][j][0] * inv, o_acc[b][j][1] * inv),
                                 T::pack(o_acc[b][j][2] * inv, o_acc[b][j][3] * inv)};
                *reinterpret_cast<u32x2*>(orow + 16 * b) = w;
            }
            if (c.lse && lg == 0) c.lse[stat_at[j]] = l == 0.f ? -INFINITY : m_run[j] + log2f(l);
        }
    }
}

// A split row: m = max over its parts, w = 2^(m_part - m), o = sum w o_part /
// sum w l_part. One wave per row; bound by reading the partial results.
template <class T, int D, bool kPaged>
__global__ __launch_bounds__(256) void window_combine_kernel(WindowCall c) {
    const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= c.rows) return;
    const int lane = threadIdx.x & 63;
    int64_t out_at;
    if constexpr (kPaged) {
        const int token = static_cast<int>(row / c.heads), head = static_cast<int>(row - int64_t(token) * c.heads);
        // Rows before the first sequence and behind the last stay as they were.
        if (token < c.offsets[0] || token >= c.offsets[c.batch]) return;
        out_at = head * c.out_rows.head + int64_t(token) * c.out_rows.token;
    } else {
        const int64_t bh = row / c.tokens, token = row - bh * c.tokens, b = bh / c.heads, head = bh - b * c.heads;
        out_at = b * c.out_rows.batch + head * c.out_rows.head + token * c.out_rows.token;
    }
    float m = -INFINITY;
    for (int p = 0; p < c.parts; ++p) m = fmaxf(m, c.partial_stat[p * c.rows + row].x);
    float l = 0.f, o[D / 64] = {};
    for (int p = 0; p < c.parts; ++p) {
        const float2 stat = c.partial_stat[p * c.rows + row];
        if (stat.y == 0.f) continue;
        const float w = fast_exp2(stat.x - m);
        l += w * stat.y;
        const float* src = c.partial_o + (p * c.rows + row) * D + lane * (D / 64);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) o[i] += w * src[i];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t* dst = static_cast<uint16_t*>(c.out) + out_at + lane * (D / 64);
    if constexpr (D == 128)
        *reinterpret_cast<uint32_t*>(dst) = T::pack(o[0] * inv, o[1] * inv);
    else
        *dst = static_cast<uint16_t>(T::pack(o[0] * inv, 0.f));
    if (c.lse && lane == 0) c.lse[row] = l == 0.f ? -INFINITY : m + log2f(l);
}

template <class T, int D, bool kPaged>
int launch_as(const WindowCall& c, hipStream_t stream) {
    const int64_t tiles = window_tiles(c), heads = kPaged ? c.kv_heads : int64_t(c.batch) * c.heads;
    const dim3 grid(window_grid(heads, tiles), static_cast<unsigned>(c.parts));
    if (c.parts == 1) {
        hipLaunchKernelGGL((window_kernel<T, D, kPaged, false>), grid, dim3(kWindowThreads), 0, stream, c, int(tiles));
        return check_launch("window_kernel");
    }
    hipLaunchKernelGGL((window_kernel<T, D, kPaged, true>), grid, dim3(kWindowThreads), 0, stream, c, int(tiles));
    if (int rc = check_launch("window_kernel")) return rc;
    hipLaunchKernelGGL((window_combine_kernel<T, D, kPaged>), dim3(static_cast<unsigned>((c.rows + 3) / 4)), dim3(256), 0, stream, c);
    return check_launch("window_combine_kernel");
}
}  // namespace

// Tiles of rows of one head (of one K/V head over a cache, in slots).
int64_t window_tiles(const WindowCall& c) {
    if (c.paged) return int64_t(c.tokens) * c.group.d / kWindowRows + c.batch;
    return (int64_t(c.tokens) + kWindowRows - 1) / kWindowRows;
}

// Parts that the keys of every tile of rows are split into: as many as give
// each CU two workgroups, with at least 8 tiles of keys in each.
int window_parts(const WindowCall& c, int64_t most_keys) {
    int64_t units = window_tiles(c) * (c.paged ? c.kv_heads : int64_t(c.batch) * c.heads);
    const int64_t key_tiles = (most_keys + kWindowKeys - 1) / kWindowKeys;
    const int64_t parts = std::min<int64_t>({(512 + units - 1) / units, key_tiles / 8, 64});
    return static_cast<int>(std::max<int64_t>(parts, 1));
}

int launch_window(const WindowCall& c, hipStream_t stream) {
    auto typed = [&](auto t) {
        using T = decltype(t);
        if (c.dim == 128) return c.paged ? launch_as<T, 128, true>(c, stream) : launch_as<T, 128, false>(c, stream);
        return c.paged ? launch_as<T, 64, true>(c, stream) : launch_as<T, 64, false>(c, stream);
    };
    return c.half ? typed(F16{}) : typed(Bf16{});
}

}  // namespace ab
