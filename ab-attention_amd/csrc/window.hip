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
// some of its rows see: the sinks' tiles, then the window's; only tiles that some
// row of a wave sees in part are masked. K and V go straight from memory into two
// rings of four LDS stages, three to five tiles ahead, through buffers that end
// where the visible keys of a tensor or a page do: what lies behind arrives as
// zeros and is never read. The step is software-pipelined: the first product of the
// next tile beside this tile's exponentials, this tile's second product beside the
// next one's logits. The reference of a row moves only where a logit (base 2) passes
// it by more than 8. P is rounded to the input type for the second product, which the
// matrix cores multiply in (the output is 2.3e-3 off in bf16 where its own rounding
// leaves 1.7e-3, in fp16 2.7e-4 and 2.1e-4; what the rounding takes would be a third
// product), the output once at the end; sums are float32. For a backward pass the
// output is known better: out + out_rest is the sum before its rounding, over the sum
// of the rounded P, whose weights add up to one again (a row that one key carries owes
// nothing to P's rounding).
//
// What bounds it: with many keys the matrix cores at the board's power limit, with
// the LDS (16 KiB read by each wave of a step) and the vector units (118
// instructions beside 32 MFMAs) close behind: 12 heads of 32,760 tokens that all see
// each other 1,130 TFLOP/s, causal over frames with a window of four 946 (rows that
// straddle frames; filling and emptying the pipelines, 9 us of each of four rounds of
// 512 workgroups, 21 us of a lone one with its launch). The straightforward form of
// this kernel (two stages, one tile at a time) did 605. With single tokens over long
// caches it is memory: 4.7 TB/s of the 4.9 that a copy reaches, the keys split over
// workgroups. 9 tiles of a short call take 14 us, half of them the pipeline's filling.
#include <algorithm>
#include <initializer_list>

#include "window.hpp"

namespace ab {
namespace {

constexpr int kRing = 4;         // stages of K and of V in LDS
// Base 2: how far a row's reference is below its largest logit when it is moved, and
// the largest logit above it, so how large P is. Thousands of weights far below the
// largest one (a sink that takes nearly all of it) add up, and below 2^-14 fp16 has
// fewer bits: there P reaches up to 2^15.9, which keeps all bits of weights down to
// 2^-22 of the largest and takes at most 2^-33 of it from any. The reference moves
// about as often as with bf16's slack of 8 (fp16 480p case 1,515 to 1,517 us; 11 below
// and a slack of 4 are 1,571).
template <class T>
constexpr float kBelow = T::kLift > 0 ? 8.0f : 0.0f;
template <class T>
constexpr float kSlack = T::kLift > 0 ? 15.9f : 8.0f;

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
__device__ __forceinline__ bool window_unit(const WindowCall& c, const WindowGrid& grid, uint32_t id, WindowUnit& u) {
    int head;
    if constexpr (!kPaged) {
        grid.place(id, head, u.tile);
        u.b = head / c.heads;
        u.head = head - u.b * c.heads;
        u.kv_head = u.head / static_cast<int>(c.group.d);
        u.n = c.tokens;
        u.off = 0;
        u.first = 0;
        u.length = c.lengths ? min(max(c.lengths[u.b], 0), c.tokens) : c.tokens;
        return true;
    } else {
        int head, slot;
        const int lane = threadIdx.x & 63;
        const int group = static_cast<int>(c.group.d), tokens = c.tokens;
        if (c.batch <= 64) {
            // Lane b looks at sequence b. The tiles of the sequences with the most
            // visible keys come first, over all heads: each adds up the tiles of those
            // before it (12 sequences of 1 to 1,111 new tokens over 1,668 to 9,000: 383
            // us in the order of their rows, 303 so).
            slot = id / c.kv_heads;
            head = id - slot * c.kv_heads;
            const int b = min(lane, c.batch - 1);
            const int off = min(max(c.offsets[b], 0), tokens), n = lane < c.batch ? min(max(c.offsets[b + 1], 0), tokens) - off : 0;
            const int tiles = n > 0 ? static_cast<int>((int64_t(n) * group + kWindowRows - 1) / kWindowRows) : 0;
            const int length = static_cast<int>(min(int64_t(max(c.lengths[b], 0)), int64_t(c.table_width) * c.page.d));
            const int cost = n > 0 ? static_cast<int>(min(int64_t(length), int64_t(c.mask.back) + c.mask.frame.d + c.mask.sinks)) : -1;
            int start = 0;
            for (int j = 0; j < c.batch; ++j) {
                const int other = __builtin_amdgcn_readlane(cost, j), its = __builtin_amdgcn_readlane(tiles, j);
                start += other > cost || (other == cost && j < lane) ? its : 0;
            }
            const uint64_t mine = __ballot(slot >= start && slot < start + tiles);
            if (mine == 0) return false;
            u.b = __builtin_amdgcn_readfirstlane(__builtin_ctzll(mine));
            u.off = __builtin_amdgcn_readlane(off, u.b);
            u.n = __builtin_amdgcn_readlane(n, u.b);
            u.length = __builtin_amdgcn_readlane(length, u.b);
            u.tile = __builtin_amdgcn_readlane(start + tiles - 1, u.b) - slot;
        } else {
            // Sequence b's tiles take the slots from offsets[b] * group / 128 + b on:
            // never fewer than it needs, so no sum over the sequences is wanted, nor a
            // lane for each of them. Not the longest first: 64 sequences of 1 to 400 new
            // tokens over up to 8,000 take 535 us as above, 601 with an empty 65th; single
            // tokens over up to 16,000 457 and 451.
            grid.place(id, head, slot);
            int before = 0;
            for (int at = 0; at < c.batch; at += 64) {
                const int b = min(at + lane, c.batch - 1);
                const int64_t start = int64_t(min(max(c.offsets[b], 0), tokens)) * group / kWindowRows + b;
                before += __popcll(__ballot(at + lane < c.batch && start <= slot));
            }
            u.b = __builtin_amdgcn_readfirstlane(before) - 1;
            if (u.b < 0) return false;
            u.off = min(max(c.offsets[u.b], 0), tokens);
            u.n = min(max(c.offsets[u.b + 1], 0), tokens) - u.off;
            u.tile = slot - static_cast<int>(int64_t(u.off) * group / kWindowRows + u.b);
            // A tile before the sequence's first: offsets that do not ascend.
            if (u.tile < 0 || int64_t(u.tile) * kWindowRows >= int64_t(u.n) * group) return false;
            u.length = static_cast<int>(min(int64_t(max(c.lengths[u.b], 0)), int64_t(c.table_width) * c.page.d));
        }
        for (int* p : {&u.off, &u.n, &u.length, &u.tile, &head}) *p = __builtin_amdgcn_readfirstlane(*p);
        u.kv_head = head;
        u.head = head * group;
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
    static constexpr int kVRing = kRing * kBytes;
    static constexpr int kVotes = 2 * kRing * kBytes;
    static constexpr int kLdsBytes = kVotes + 16;
};

// What `rounded` lacks of two values, rounded itself (nothing of values that are not
// finite).
template <class T>
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t rounded) {
    const float x = a - T::lo(rounded), y = b - T::hi(rounded);
    return T::pack(fabsf(x) < INFINITY ? x : 0.f, fabsf(y) < INFINITY ? y : 0.f);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// v_max_f32 without the NaN quieting that the compiler adds around fmaxf.
__device__ __forceinline__ float vmax(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
#pragma clang diagnostic pop

// The maxima of a and b over the four lanes l, 16 + l, 32 + l, 48 + l.
__device__ __forceinline__ void max_over_rows(float& a, float& b) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    const float m = vmax(__uint_as_float(s[0]), __uint_as_float(s[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    const float m2 = vmax(__uint_as_float(t[0]), __uint_as_float(t[1]));
    const auto u = __builtin_amdgcn_permlane16_swap(__float_as_uint(m2), __float_as_uint(m2), false, false);
    a = __uint_as_float(u[0]);
    b = __uint_as_float(u[1]);
}

template <class T, int D, bool kPaged, bool kSplit>
__global__ __launch_bounds__(kWindowThreads, 2) void window_kernel(WindowCall c, WindowGrid places) {
    using Tile = WindowTile<T, D>;
    constexpr int kSteps = Tile::kSteps, kBlocks = Tile::kBlocks, kOps = Tile::kOps;
    extern __shared__ __align__(16) unsigned char smem[];
    touch(c.q, c.k_rows.batch, c.row.batch, c.lengths, c.rows, places.heads);

    WindowUnit u;
    if (!window_unit<kPaged>(c, places, blockIdx.x, u)) return;
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
    // Row 16j + li of this wave's 32: its token and query head.
    auto row_of = [&](int j, int& token, int& head) {
        const int r = wave * 32 + 16 * j + li, packed = row0 + min(r, rows - 1);
        token = kPaged ? packed / group : packed;
        head = u.head + (kPaged ? packed - token * group : 0);
        return r < rows;
    };

    // Q as the B operand of S^T = K Q^T: row 16j + li, dims 32s + 8lg .. + 7. The
    // row's own bounds; all zero for a row without keys.
    u32x4 bq[2][kSteps];
    auto read_q = [&]() {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            int token, head;
            row_of(j, token, head);
            const uint16_t* qrow = static_cast<const uint16_t*>(c.q) + u.b * c.q_rows.batch + head * c.q_rows.head +
                                   int64_t(u.off + token) * c.q_rows.token + 8 * lg;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) bq[j][s] = *reinterpret_cast<const u32x4*>(qrow + 32 * s);
        }
    };
    int low[2], seen[2], sink[2];  // keys low .. low + seen - 1 and 0 .. sink - 1
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        int token, head;
        const bool stored = row_of(j, token, head);
        const int p = u.first + token;
        const bool sees = stored && p >= 0 && p < u.length;
        const int high = mask.high(max(p, 0), u.length);
        low[j] = mask.low(max(p, 0));
        seen[j] = sees ? high - low[j] : 0;
        sink[j] = sees ? min(mask.sinks, high) : 0;
    }
    // Tiles that every row of this wave sees need no mask: keys from full_low to
    // full_high, and those before full_sink. A wave with a row that exists but
    // sees nothing masks every tile.
    int full_low = 0, full_high = 0, full_sink = 0;
    const int wave_rows = min(32, rows - wave * 32);
    const bool active = wave_rows > 0;
    if (active) {
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
    const int last_entry = c.table_width - 1;

    // Whether a key that some row would see lies on no page (then every tile
    // asks the table for its keys). Pages between the sinks and the window, which
    // may have been given back, do not count.
    bool holes = false;
    if constexpr (kPaged) {
        bool bad = false;
        auto scan = [&](int from, int to) {
            const int page = static_cast<int>(c.page.d);
            for (int i = from / page + tid; from < to && i <= (to - 1) / page; i += kWindowThreads)
                bad |= static_cast<uint32_t>(table[i]) >= static_cast<uint32_t>(c.pages);
        };
        if (tiles > 0) {
            const int last = tile0 + tiles - 1;
            if (tile0 < range.sink_tiles) {
                // The window may begin in the sinks' last tile.
                const int from = range.key(tile0), to = min(kWindowKeys * min(last + 1, range.sink_tiles), end);
                scan(from, min(mask.sinks, to));
                scan(max(mask.low(p_first), from), to);
            }
            if (last >= range.sink_tiles) scan(range.key(max(tile0, range.sink_tiles)), min(range.key(last) + kWindowKeys, end));
        }
        uint32_t* votes = reinterpret_cast<uint32_t*>(smem + Tile::kVotes);
        const uint32_t vote = __any(bad) ? 1u : 0u;
        if (lane == 0) votes[wave] = vote;
        landed_and_barrier<0>();
        const u32x4 all = *reinterpret_cast<const u32x4*>(votes);
        holes = __builtin_amdgcn_readfirstlane(all[0] | all[1] | all[2] | all[3]) != 0;
    }
    auto on_page = [&](int key) {
        const uint32_t q0 = __umulhi(static_cast<uint32_t>(key), c.page.m);
        const uint32_t index = q0 + (static_cast<uint32_t>(key) - q0 * c.page.d >= c.page.d ? 1u : 0u);
        return key < end && static_cast<uint32_t>(table[min(index, static_cast<uint32_t>(c.table_width - 1))]) < static_cast<uint32_t>(c.pages);
    };

    // Transfers of this wave: keys 8w .. 8w + 7 of a tile, kOpKeys at a time.
    // K keeps rows of D elements whose 16-byte chunks are swizzled (position =
    // chunk ^ key); V keeps, for every four keys, blocks of 4 keys x 16 dims,
    // block m at position m ^ (quad & 1): both the row reads of K and the
    // transposing reads of V then spread over the banks.
    uint32_t k_src[kOps], v_src[kOps];
#pragma unroll
    for (int e = 0; e < kOps; ++e) {
        constexpr int kChunks = D / 8;
        const int key = lane / kChunks, pos = lane % kChunks, in_tile = 8 * wave + Tile::kOpKeys * e + key;
        k_src[e] = uint32_t(Tile::kOpKeys * e + key) * k_token + uint32_t(pos ^ (in_tile % kChunks)) * 16u;
        const int quad = D == 128 ? e : lane >> 5, block = (lane >> 3) % kBlocks, r = (lane >> 1) & 3, h = lane & 1;
        v_src[e] = uint32_t(4 * quad + r) * v_token + uint32_t(2 * (block ^ (quad & 1)) + h) * 16u;
    }
    // Where this wave's eight keys of a tile lie: the page, the first key's place in
    // it, and how many of the page's (or tensor's) keys exist. Nothing for tiles
    // past the last one (their transfers only keep the count of each step) and for
    // keys that lie on no page.
    struct Place {
        int32_t page;
        uint32_t at, there;
    };
    // The next place: its tile, its first key, and over a cache the page table's
    // entry, which ask() fetches well before next_place() takes it.
    int next_tile = 0, next_key = 0, next_entry = -1;
    uint32_t next_at = 0;
    auto ask = [&]() {
        if constexpr (kPaged) {
            const uint32_t key = next_key + 8 * wave;
            const uint32_t near = __umulhi(key, c.page.m), rest = key - near * c.page.d;
            const uint32_t index = rest >= c.page.d ? near + 1 : near;
            next_at = rest >= c.page.d ? rest - c.page.d : rest;
            const auto entries = (const __attribute__((address_space(4))) int32_t*)reinterpret_cast<uintptr_t>(table);
            next_entry = entries[min(index, static_cast<uint32_t>(last_entry))];
        }
    };
    auto first_place = [&]() {
        next_tile = 0;
        next_key = range.key(tile0);
    };
    auto next_place = [&]() {
        const int key = next_key + 8 * wave;
        const bool there = next_tile < tiles;
        Place p{0, static_cast<uint32_t>(key), there ? static_cast<uint32_t>(end) : 0u};
        if constexpr (kPaged) {
            const bool is_page = there && key < end && static_cast<uint32_t>(next_entry) < static_cast<uint32_t>(c.pages);
            p.page = is_page ? next_entry : 0;
            p.at = next_at;
            p.there = is_page ? min(c.page.d, static_cast<uint32_t>(end - key) + next_at) : 0u;
        }
        ++next_tile;
        next_key = tile0 + next_tile == range.sink_tiles ? range.window : next_key + kWindowKeys;
        return p;
    };
    auto ask_place = [&]() {
        ask();
        return next_place();
    };
    // n rows take n * token - less bytes (kept from the compiler, which turns the sum
    // into a borrow in vector registers).
    uint32_t k_less = k_token - 2 * D, v_less = v_token - 2 * D;
    asm volatile("" : "+s"(k_less), "+s"(v_less));
    const uint32_t k_all = end * k_token - k_less, v_all = end * v_token - v_less;
    auto move = [&](const char* base, const Rows& rows_of, uint32_t token, uint32_t less, uint32_t all, const uint32_t (&src)[kOps],
                    const Place& p, uint32_t lds) {
        const u32x4 buffer = buffer_of(base + (kPaged ? int64_t(p.page) * rows_of.batch * 2 : 0),
                                       p.there == 0 ? 0 : kPaged ? p.there * token - less : all);
        const uint32_t at = p.at * token;
        if constexpr (kOps == 2)
            buffer_to_lds(buffer, src[0] + at, src[1] + at, lds + wave * (8 * D * 2));
        else
            buffer_to_lds(buffer, src[0] + at, lds + wave * (8 * D * 2));
    };
    auto move_k = [&](int t, const Place& p) {
        move(kbase, c.k_rows, k_token, k_less, k_all, k_src, p, lds0 + (t & (kRing - 1)) * Tile::kBytes);
    };
    auto move_v = [&](int t, const Place& p) {
        move(vbase, c.v_rows, v_token, v_less, v_all, v_src, p, lds0 + Tile::kVRing + (t & (kRing - 1)) * Tile::kBytes);
    };

    // Reads of operands: K's row 16h + li, chunk 4s + lg; V's quad lg + 4h, block
    // b, of which lane li gets dim 16b + li of the four keys.
    uint32_t k_abs[kSteps], v_abs[2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) k_abs[s] = lds0 + li * (2 * D) + 16 * ((4 * s + lg) ^ (li % (D / 8)));
    {
        const int par = lg & 1, base = Tile::kVRing + lg * Tile::kQuadBytes + 32 * (li >> 2) + 8 * (li & 3);
        v_abs[0] = lds0 + base + par * 128;  // even block: position block + par
        v_abs[1] = lds0 + base - par * 128;  // odd block: position block - par
    }
    auto read_k = [&](int t, int f) {  // f = kSteps h + s
        return lds_read16(k_abs[f % kSteps] + (t & (kRing - 1)) * Tile::kBytes + (f / kSteps) * 16 * 2 * D);
    };
    auto read_v = [&](int t, int b, int h) {
        return lds_read_transposed(v_abs[b & 1] + (t & (kRing - 1)) * Tile::kBytes + b * 128 + h * 4 * Tile::kQuadBytes);
    };
    // Tiles without a mask: `clear` of them from `clear_from` on, and those before
    // clear_sink.
    int clear_from = 0, clear = 0, clear_sink = 0;
    if (!holes) {
        const int skipped = range.sink_tiles - tile0;  // tiles of this part before the window's
        clear_from = max(skipped, 0) + max(0, full_low - range.window - max(-skipped, 0) * kWindowKeys + kWindowKeys - 1) / kWindowKeys;
        clear = max(0, min(tiles, (full_high - range.window) / kWindowKeys + skipped) - clear_from);
        clear_sink = min(range.sink_tiles ? skipped : tiles, full_sink / kWindowKeys - tile0);
    }
    auto is_masked = [&](int t) {
        return static_cast<uint32_t>(t - clear_from) >= static_cast<uint32_t>(clear) && t >= clear_sink;
    };
    // Bit r of the result: key 16h + 4lg + r of tile t is seen by row 16j + li.
    auto seen_keys = [&](int t, int h, int j) {
        const int key = range.key(tile0 + t) + 16 * h + 4 * lg;
        uint32_t bits = 0;
        if (t < tiles && (!kPaged || !holes || on_page(key)))
#pragma unroll
            for (int r = 0; r < 4; ++r)
                bits |= static_cast<uint32_t>(key + r - low[j]) < static_cast<uint32_t>(seen[j]) || key + r < sink[j] ? 1u << r : 0u;
        return bits;
    };

    f32x4 o_acc[kBlocks][2];  // dims 16b + 4lg .. + 3 of row 16j + li
    // Reference of row j, sum of its weights, for out_rest the same of the rounded ones;
    // -inf until the row's first finite logit, then kSlack.
    float m_run[2], l_run[2], r_run[2], slack[2];
    auto reset = [&]() {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) o_acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            m_run[j] = 0.f;
            l_run[j] = r_run[j] = 0.f;
            slack[j] = -INFINITY;
        }
    };
    auto start_s = [&](const u32x4 (&ka)[2 * kSteps], f32x4 (&s)[4]) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4 * kSteps; ++x) {
            const int step = x >> 2, h = (x >> 1) & 1, j = x & 1;
            s[2 * h + j] = T::mfma16(ka[kSteps * h + step], bq[j][step], s[2 * h + j]);
        }
    };
    // Logits of tile t against the rows' references, from S; mx[j] their maximum
    // over this lane's keys.
    auto mask_logits = [&](int t, f32x4 (&s)[4], float (&mx)[2]) {
        mx[0] = mx[1] = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t bits = seen_keys(t, h, j);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (!(bits >> r & 1)) s[2 * h + j][r] = -INFINITY;
                    mx[j] = fmaxf(mx[j], s[2 * h + j][r]);
                }
            }
    };
    // Moves the reference of the rows whose maximum has risen more than kSlack above
    // it (or that have none yet): their sums, and the logits at hand, follow.
    auto move_reference = [&](f32x4 (&s)[4], float (&mx)[2]) {
        // A lane's own keys show it: no exchange while nothing grows.
        if (!__any(mx[0] > slack[0] || mx[1] > slack[1])) return;
        max_over_rows(mx[0], mx[1]);
        const bool grow0 = mx[0] > slack[0], grow1 = mx[1] > slack[1];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bool grow = j ? grow1 : grow0;
            const float shift = grow ? mx[j] - kBelow<T> : 0.f;
            const float alpha = slack[j] == kSlack<T> ? fast_exp2(-shift) : 1.f;  // the sums are 0 before
            slack[j] = grow ? kSlack<T> : slack[j];
            m_run[j] += shift;
            l_run[j] *= alpha;
            r_run[j] *= alpha;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) o_acc[b][j] *= alpha;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[2 * h + j][r] -= shift;
        }
    };

    // The pass that calls take. Step t: phase A computes S(t + 1) beside p = 2^y of
    // tile t, the reads of V(t) and the transfers of K(t + 5) and V(t + 3); phase B
    // adds V(t)^T P(t)^T beside the logits of tile t + 1 and the reads of K(t + 2).
    // Returns whether a tile that some rows see in part held a value that is not
    // finite: 0 times it is no zero, so the tile cannot be computed like that.
    auto fast_pass = [&]() -> bool {
        uint32_t odd = 0;
        // Places of K(t + 5), of tile t + 4 and of V(t + 3) before step t.
        Place kp, mp, vp;
        auto next_step = [&]() {
            vp = mp;
            mp = kp;
            kp = next_place();
        };
        auto step = [&](int t, f32x4 (&sc)[4], f32x4 (&sn)[4], float (&mx)[2], u32x4 (&ka)[2 * kSteps]) {
            landed_and_barrier<4 * kOps>();
            ask();
            if (!active) {
                move_k(t + 5, kp);
                move_v(t + 3, vp);
                next_step();
                return;
            }
            move_reference(sc, mx);
            constexpr int kEach = 16 / (4 * kSteps);  // values of P beside each MFMA
            uint32_t pw[2][4];
            float psum[2] = {0.f, 0.f}, p_prev = 0.f;
            u32x4 va[kBlocks];
            i16x4 v_lo = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 4; ++x) sn[x] = f32x4{0.f, 0.f, 0.f, 0.f};
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < 4 * kSteps; ++x) {
                const int st = x >> 2, h = (x >> 1) & 1, j = x & 1;
                sn[2 * h + j] = T::mfma16(ka[kSteps * h + st], bq[j][st], sn[2 * h + j]);
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int e = x * kEach + i, n = e >> 2, r = e & 3;  // n = 2h' + j'
                    const float p = fast_exp2(sc[n][r]);
                    psum[n & 1] += p;
                    if (e & 1) pw[n & 1][2 * (n >> 1) + (r >> 1)] = T::pack(p_prev, p);
                    p_prev = p;
                }
                const i16x4 vh = read_v(t, x >> 1, x & 1);
                if (x & 1) va[x >> 1] = __builtin_bit_cast(u32x4, __builtin_shufflevector(v_lo, vh, 0, 1, 2, 3, 4, 5, 6, 7));
                else v_lo = vh;
                if (x == 2) move_k(t + 5, kp);
                if (x == 6) move_v(t + 3, vp);
                __builtin_amdgcn_sched_barrier(0);
            }
            // P is made here, beside the MFMAs, and not moved behind the branch.
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(pw[i >> 2][i & 3]));
            asm volatile("" : "+v"(psum[0]), "+v"(psum[1]));
            l_run[0] += psum[0];
            l_run[1] += psum[1];
            if constexpr (!kPaged)
                if (c.out_rest)
#pragma unroll
                    for (int i = 0; i < 8; ++i) r_run[i >> 2] = T::add(pw[i >> 2][i & 3], r_run[i >> 2]);
            if (is_masked(t)) {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int w = 0; w < 4; ++w) odd |= (va[b][w] & T::kExponent) + T::kOverflow;
            }
            mx[0] = mx[1] = -INFINITY;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int x = 0; x < 2 * kBlocks; ++x) {
                const int b = x >> 1, j = x & 1;
                const u32x4 p = {pw[j][0], pw[j][1], pw[j][2], pw[j][3]};
                o_acc[b][j] = T::mfma16(va[b], p, o_acc[b][j]);
                if (x < 2 * kSteps) ka[x] = read_k(t + 2, x);
                constexpr int kPairs = 8 / kBlocks;  // pairs of logits of tile t + 1 beside every second MFMA
                if (x & 1)
#pragma unroll
                    for (int i = 0; i < kPairs; ++i) {
                        const int e = 2 * ((x >> 1) * kPairs + i), n = e >> 2, r = e & 3;
                        const float y0 = __builtin_fmaf(sn[n][r], c.scale_log2, -m_run[n & 1]);
                        const float y1 = __builtin_fmaf(sn[n][r + 1], c.scale_log2, -m_run[n & 1]);
                        sn[n][r] = y0;
                        sn[n][r + 1] = y1;
                        mx[n & 1] = fmaxf(fmaxf(mx[n & 1], y0), y1);
                    }
                if (x == 2 * kBlocks - 4) next_step();
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(mx[0]), "+v"(mx[1]));  // made beside the MFMAs too
            if (is_masked(t + 1)) mask_logits(t + 1, sn, mx);
        };

        // K(0 .. 3) and V(0 .. 2); S(0) and K(1) to registers once K(0) and K(1) are
        // in; K(4) goes to K(0)'s place only after every wave has read that. The last
        // transfers before step 0 are then K(3), V(1), V(2), K(4), as its wait expects.
        {
            first_place();
            const Place p0 = ask_place(), p1 = ask_place(), p2 = ask_place();
            vp = ask_place();
            move_k(0, p0);
            move_k(1, p1);
            move_k(2, p2);
            move_v(0, p0);
            move_k(3, vp);
            move_v(1, p1);
            move_v(2, p2);
        }
        if (active) read_q();  // behind the transfers, not before them
        mp = ask_place();
        kp = ask_place();
        f32x4 s0[4], s1[4];
        u32x4 ka[2 * kSteps];
        float mx[2] = {-INFINITY, -INFINITY};
        landed_and_barrier<5 * kOps>();
        if (active) {
#pragma unroll
            for (int f = 0; f < 2 * kSteps; ++f) ka[f] = read_k(0, f);
            start_s(ka, s0);
#pragma unroll
            for (int f = 0; f < 2 * kSteps; ++f) ka[f] = read_k(1, f);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s0[n][r] *= c.scale_log2;
                    mx[n & 1] = fmaxf(mx[n & 1], s0[n][r]);
                }
            if (is_masked(0)) mask_logits(0, s0, mx);
        }
        // Every wave's reads of K(0) are done. Q, asked for last, is here, and with it
        // all transfers; said to the compiler too, which else waits for Q in the loop.
        landed_and_barrier<0>();
        move_k(4, mp);
        int t = 0;
        for (; t + 3 < tiles; t += 4) {
            step(t, s0, s1, mx, ka);
            step(t + 1, s1, s0, mx, ka);
            step(t + 2, s0, s1, mx, ka);
            step(t + 3, s1, s0, mx, ka);
        }
        for (; t + 1 < tiles; t += 2) {
            step(t, s0, s1, mx, ka);
            step(t + 1, s1, s0, mx, ka);
        }
        if (t < tiles) step(t, s0, s1, mx, ka);
        // No transfer may still be landing when the LDS is released or filled again.
        uint32_t* votes = reinterpret_cast<uint32_t*>(smem + Tile::kVotes);
        const uint32_t vote = __any((odd & 0x80008000u) != 0) ? 1u : 0u;
        landed_and_barrier<0>();
        if (lane == 0) votes[wave] = vote;
        landed_and_barrier<0>();
        const u32x4 all = *reinterpret_cast<const u32x4*>(votes);
        return __builtin_amdgcn_readfirstlane(all[0] | all[1] | all[2] | all[3]) != 0;
    };

    // The same sums, tile by tile, with values that are not finite kept from the
    // rows that do not see them: V without them, and where a row sees one, an
    // infinity of its sign (or, for NaN, of both).
    auto careful_pass = [&]() {
        reset();
        landed_and_barrier<0>();
        first_place();
        for (int t = 0; t < tiles; ++t) {
            const Place p = ask_place();
            move_k(0, p);
            move_v(0, p);
            landed_and_barrier<0>();
            if (active) {
                u32x4 ka[2 * kSteps];
                f32x4 s[4];
                float mx[2];
#pragma unroll
                for (int f = 0; f < 2 * kSteps; ++f) ka[f] = read_k(0, f);
                start_s(ka, s);
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[n][r] = __builtin_fmaf(s[n][r], c.scale_log2, -m_run[n & 1]);
                mask_logits(t, s, mx);
                move_reference(s, mx);
                u32x4 pw[2], sees[2];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t bits = seen_keys(t, n >> 1, n & 1);
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const float a = fast_exp2(s[n][r]), b = fast_exp2(s[n][r + 1]);
                        l_run[n & 1] += a + b;
                        pw[n & 1][2 * (n >> 1) + r / 2] = T::pack(a, b);
                        r_run[n & 1] = T::add(pw[n & 1][2 * (n >> 1) + r / 2], r_run[n & 1]);
                        sees[n & 1][2 * (n >> 1) + r / 2] = (bits >> r & 1 ? T::kOne : 0u) | (bits >> (r + 1) & 1 ? T::kOne << 16 : 0u);
                    }
                }
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const u32x4 a = __builtin_bit_cast(u32x4, __builtin_shufflevector(read_v(0, b, 0), read_v(0, b, 1), 0, 1, 2, 3, 4, 5, 6, 7));
                    u32x4 finite, up, down;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        // All ones in the halves that are no number, are NaN, are negative.
                        const uint32_t none = ((((a[w] & T::kExponent) + T::kOverflow) & 0x80008000u) >> 15) * 0xffffu;
                        const uint32_t nan = ((((a[w] & ~T::kExponent & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u) >> 15) * 0xffffu;
                        const uint32_t minus = ((a[w] & 0x80008000u) >> 15) * 0xffffu;
                        finite[w] = a[w] & ~none;
                        up[w] = none & (nan | ~minus) & (T::kOne * 0x10001u);
                        down[w] = none & (nan | minus) & (T::kOne * 0x10001u);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                        const f32x4 ups = T::mfma16(up, sees[j], zero), downs = T::mfma16(down, sees[j], zero);
                        o_acc[b][j] = T::mfma16(finite, pw[j], o_acc[b][j]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            o_acc[b][j][r] += ups[r] > 0.f ? INFINITY : 0.f;
                            o_acc[b][j][r] -= downs[r] > 0.f ? INFINITY : 0.f;
                        }
                    }
                }
            }
            landed_and_barrier<0>();  // read before the next tile's transfers
        }
    };
    // Without a key there may be no page table either: nothing is asked for.
    reset();
    if (tiles > 0 && fast_pass()) careful_pass();

    if (!active) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        auto over_rows = [](float x) {  // the sum over the four lanes of a row
            const auto s16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            const float y = __uint_as_float(s16[0]) + __uint_as_float(s16[1]);
            const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
            return __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
        };
        const float l = over_rows(l_run[j]), rounded = over_rows(r_run[j]);
        int token, head;
        if (!row_of(j, token, head)) continue;
        const int64_t stat_at = u.b * c.row.batch + head * c.row.head + int64_t(u.off + token) * c.row.token;
        if constexpr (kSplit) {
            const int64_t at = blockIdx.y * c.rows + stat_at;
            if (lg == 0) {
                c.partial_stat[at] = float2{slack[j] == kSlack<T> ? m_run[j] : -INFINITY, l};
                if (!kPaged && c.out_rest) c.partial_rounded[at] = rounded;
            }
            if (l == 0.f) continue;
            float* dst = c.partial_o + at * D + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4*>(dst + 16 * b) = o_acc[b][j];
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l, better = kPaged || rounded == 0.f ? inv : 1.0f / rounded;
            uint16_t* orow = static_cast<uint16_t*>(c.out) + u.b * c.out_rows.batch + head * c.out_rows.head +
                             int64_t(u.off + token) * c.out_rows.token + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const f32x4 o = o_acc[b][j] * inv;
                const u32x2 w = {T::pack(o[0], o[1]), T::pack(o[2], o[3])};
                *reinterpret_cast<u32x2*>(orow + 16 * b) = w;
                if (c.out_rest) {
                    const f32x4 before = o_acc[b][j] * better;
                    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(c.out_rest) + (orow - static_cast<uint16_t*>(c.out)) + 16 * b) =
                        u32x2{rest_of<T>(before[0], before[1], w[0]), rest_of<T>(before[2], before[3], w[1])};
                }
            }
            if (c.lse && lg == 0) c.lse[stat_at] = l == 0.f ? -INFINITY : m_run[j] + log2f(l);
        }
    }
}

// A split row: m = max over its parts, w = 2^(m_part - m), o = sum w o_part /
// sum w l_part. One wave per row: lane p looks at part p (of at most 64), then all
// lanes add up the parts' rows, four loads ahead. Bound by reading the partial
// results or, for few rows, by two loads after one another (part after part, 52 parts
// took 50 us).
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
    float2 stat = {-INFINITY, 0.f};
    float rounded = 0.f;
    if (lane < c.parts) {
        stat = c.partial_stat[lane * c.rows + row];
        if (!kPaged && c.out_rest) rounded = c.partial_rounded[lane * c.rows + row];
    }
    const bool some = stat.y != 0.f;  // a part without a key has written no row
    const uint64_t written = __ballot(some);
    float m = some ? stat.x : -INFINITY;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) m = fmaxf(m, __shfl_xor(m, s));
    const float weight = some ? fast_exp2(stat.x - m) : 0.f;
    float l = some ? weight * stat.y : 0.f, o[D / 64] = {};
    rounded = some ? weight * rounded : 0.f;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        l += __shfl_xor(l, s);
        rounded += __shfl_xor(rounded, s);
    }
    constexpr int kAhead = 4;
    for (int p0 = 0; p0 < c.parts; p0 += kAhead) {
        float x[kAhead][D / 64];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float* src = c.partial_o + (min(p0 + i, c.parts - 1) * c.rows + row) * D + lane * (D / 64);
#pragma unroll
            for (int e = 0; e < D / 64; ++e) x[i][e] = src[e];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (p0 + i >= c.parts) break;
            if (!(written >> (p0 + i) & 1)) continue;
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), p0 + i));
            // An infinite value is seen however small its part's weight is.
#pragma unroll
            for (int e = 0; e < D / 64; ++e) o[e] += w == 0.f && !(fabsf(x[i][e]) < INFINITY) ? x[i][e] : w * x[i][e];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l, better = kPaged || rounded == 0.f ? inv : 1.0f / rounded;
    const int64_t at = out_at + lane * (D / 64);
    const float first = o[0], second = D == 128 ? o[D / 64 - 1] : 0.f;
    const uint32_t w = T::pack(first * inv, second * inv), rest = rest_of<T>(first * better, second * better, w);
    auto store = [&](void* to, uint32_t value) {
        if constexpr (D == 128)
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(to) + at) = value;
        else
            static_cast<uint16_t*>(to)[at] = static_cast<uint16_t>(value);
    };
    store(c.out, w);
    if (c.out_rest) store(c.out_rest, rest);
    if (c.lse && lane == 0) c.lse[row] = l == 0.f ? -INFINITY : m + log2f(l);
}

template <class T, int D, bool kPaged>
int launch_as(const WindowCall& c, hipStream_t stream) {
    const int64_t tiles = window_tiles(c), heads = kPaged ? c.kv_heads : int64_t(c.batch) * c.heads;
    const WindowGrid places = window_grid(heads, tiles);
    const dim3 grid(places.size(), static_cast<unsigned>(c.parts));
    const auto kernel = c.parts == 1 ? window_kernel<T, D, kPaged, false> : window_kernel<T, D, kPaged, true>;
    constexpr int kLds = WindowTile<T, D>::kLdsBytes;
    if (int rc = ensure_lds_limit(reinterpret_cast<const void*>(kernel), kLds)) return rc;
    hipLaunchKernelGGL(kernel, grid, dim3(kWindowThreads), kLds, stream, c, places);
    if (int rc = check_launch("window_kernel")) return rc;
    if (c.parts == 1) return 0;
    hipLaunchKernelGGL((window_combine_kernel<T, D, kPaged>), dim3(static_cast<unsigned>((c.rows + 3) / 4)), dim3(256), 0, stream, c);
    return check_launch("window_combine_kernel");
}
}  // namespace

// Tiles of rows of one head (of one K/V head over a cache, in slots).
int64_t window_tiles(const WindowCall& c) {
    if (c.paged) return int64_t(c.tokens) * c.group.d / kWindowRows + c.batch;
    return (int64_t(c.tokens) + kWindowRows - 1) / kWindowRows;
}

// Parts that the keys of every tile of rows are split into: those that cost least.
// A workgroup's time is its steps and about 6 us to fill and empty its pipeline; a step
// takes 0.80 us where each CU has a workgroup and 0.95 where it has two (D = 64: 0.6 of
// that), and more than 512 workgroups go in rounds: a fit to whole calls, masked tiles
// among them (calls without masks: 0.64 and 0.93 us a step). Splitting adds a second kernel
// of 6 us and the partial results' traffic. Over 150 calls of 1 to 400 GFLOP drawn from
// the range of sizes this took 5.7 % less time than as many parts as give each CU two
// workgroups; lone steps of 0.55 us (the dense kernel's) took 2.6 % less, of 0.90 and
// 0.95 the same. One token of 8 heads over 16,384 keys: 31 us.
int window_parts(const WindowCall& c, int64_t most_keys) {
    const double units = double(window_tiles(c)) * (c.paged ? c.kv_heads : int64_t(c.batch) * c.heads);
    const int64_t steps = (most_keys + kWindowKeys - 1) / kWindowKeys;
    const double scale = c.dim == 128 ? 1.0 : 0.6;
    auto cost = [&](int64_t parts) {
        const double groups = units * double(parts), rounds = std::max(1.0, groups / 512);
        const double step = scale * (groups <= 256 ? 0.80 : 0.80 + 0.15 * std::min(1.0, groups / 256 - 1));
        const double traffic = double(c.rows) * (c.dim * 4.0 + 8) * double(parts) * 2 / 4.5e6;
        return rounds * (double((steps + parts - 1) / parts) * step + 6) + (parts > 1 ? 6 + traffic : 0.0);
    };
    int best = 1;
    double least = 0.95 * cost(1);
    for (int64_t parts = 2; parts <= 64 && parts * 4 <= steps; ++parts)
        if (cost(parts) < least) {
            best = static_cast<int>(parts);
            least = cost(parts);
        }
    return best;
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
