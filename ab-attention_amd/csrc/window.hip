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
//
// A tree of drafted tokens (tree_attention_kernel) takes the same passes over tiles of 128 or
// 256 rows. Its rows are not in the order of their positions: the bounds of clear tiles are
// those of all a sequence's tokens, and what each token sees of the other tiles (the ends of
// sinks and window, the drafts, all of them where a page is missing) is made into words of 32
// keys in LDS before the passes, which then take one LDS read for a masked tile and row, and
// none of the mask's arithmetic. The first form walked up the tree in every masked tile (4 x
// 701 drafts 195 us, now 82). Bound like the others: one sequence of 64 drafts, 256 rows over
// 100,000 keys, 132 to 136 us where reading takes 84 and the products 81; of 16 drafts 98, 4.2
// TB/s, of one 91; a few keys (26 drafts over 1,017) 18 us, all of it one thing after another:
// which sequence, its page table, its masks, four tiles of keys, 3,000 instructions of one wave.
// (Calls in a row, with the kernel that joins parts: 9 us of the first, 8, 4 of the last.)
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
    // Of a tree: which part of how many of the tile's keys, where its rows go if there are
    // several, and how far the next part's place is.
    int part, parts, slot, stride;
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

// x of the lane that a DPP control names, 0 where there is none.
template <int kControl>
__device__ __forceinline__ int lane_moved(int x) {
    return __builtin_amdgcn_update_dpp(0, x, kControl, 15, 15, true);
}
template <int kControl>
__device__ __forceinline__ float lane_moved(float x) {
    return __builtin_bit_cast(float, lane_moved<kControl>(__builtin_bit_cast(int, x)));
}
template <class N>
__device__ __forceinline__ N lane_value(N x, int lane) {
    return __builtin_bit_cast(N, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// x and those of the lanes before.
template <class N>
__device__ __forceinline__ N running_sum(N x, int lane) {
    x += lane_moved<0x111>(x);  // row_shr 1, 2, 4, 8
    x += lane_moved<0x112>(x);
    x += lane_moved<0x114>(x);
    x += lane_moved<0x118>(x);
    const N one = lane_value(x, 15), two = one + lane_value(x, 31), three = two + lane_value(x, 47);
    return x + (lane < 16 ? N(0) : lane < 32 ? one : lane < 48 ? two : three);
}
__device__ __forceinline__ int most_of_lanes(int x) {  // of numbers that are not negative
    x = max(x, lane_moved<0x111>(x));
    x = max(x, lane_moved<0x112>(x));
    x = max(x, lane_moved<0x114>(x));
    x = max(x, lane_moved<0x118>(x));
    return max(max(__builtin_amdgcn_readlane(x, 15), __builtin_amdgcn_readlane(x, 31)),
               max(__builtin_amdgcn_readlane(x, 47), __builtin_amdgcn_readlane(x, 63)));
}

// A kernel's first argument, read anew where it is asked for: else the compiler reads all of
// it at the start and keeps it in lanes of vector registers, two instructions for every use.
__device__ __forceinline__ const WindowCall& arguments() {
    auto at = (const __attribute__((address_space(4))) WindowCall*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const WindowCall*)at;
}

// A sequence of a tree's call: its rows' tiles, and the tiles of keys that they take.
struct TreeSequence {
    int off, n, length, tiles, steps;
};
template <int kRows>
__device__ __forceinline__ TreeSequence tree_sequence(const WindowCall& c, int b) {
    TreeSequence s;
    const bool there = b < c.batch;
    b = min(b, c.batch - 1);
    s.off = min(max(c.offsets[b], 0), c.tokens);
    s.n = there ? min(max(c.offsets[b + 1], 0), c.tokens) - s.off : 0;
    s.length = static_cast<int>(min(int64_t(max(c.lengths[b], 0)), int64_t(c.table_width) * c.page.d));
    s.tiles = s.n > 0 ? (s.n * static_cast<int>(c.group.d) + kRows - 1) / kRows : 0;
    TileRange range;
    range.set(c.mask, max(s.length - s.n, 0), s.length - 1, s.length);
    s.steps = s.tiles > 0 ? max(range.tiles, 1) : 0;  // rows that see nothing are written too
    return s;
}

// How many steps a part has at most, by what the call's sequences have: steps of all tiles of
// rows, those tiles, the longest's steps; and the parts that they have with this lane's
// tree_steps, or 0 for an estimate.
//
// How many sequences there are, and how long they are, is on the device, so the kernel
// itself deals out the work. With `steps` tiles of keys for each of the `tiles` of rows of
// a sequence, all are cut into parts of at most C steps; lane k looks at C = longest / (k + 1),
// and the C that costs least is taken: a workgroup's C steps and its filling, in rounds
// where there are more workgroups than run at once, or what reading all keys takes, if that
// is more; parts cost a second kernel and the traffic of their sums. (The same number of
// steps for every workgroup, of two tiles of rows if need be, is slower, as each tile fills
// the pipeline anew: 8 sequences of 4,026 keys 50 us, in whole parts 41.)
//
// Where a CU has one workgroup at a time (256 rows), one more than there are CUs takes a
// whole round more, so the parts are counted: in 80 calls 8 took 4 to 30 % less than by
// an estimate and fractions of a round (8 ragged sequences of 12,000 keys 85 us, 105), none
// over 4 % more. Two or three workgroups to a CU fill in for each other, and counting costs
// what it gives.
__device__ __forceinline__ float tree_steps(int longest) { return fmaxf(ceilf(longest / ((threadIdx.x & 63) + 1.f)), 1.f); }
__device__ __forceinline__ int tree_part(const WindowCall& c, float work, int units, int longest, float parts) {
    const int lane = threadIdx.x & 63, heads = c.kv_heads;
    const float steps = tree_steps(longest), whole = static_cast<float>(units) * heads;
    // Workgroups, and the most there can be.
    const float cut = work * heads / steps, most = cut + whole;
    const float groups = lane == 0 ? whole : parts > 0.f ? parts * heads : c.batch == 1 ? whole * ceilf(longest / steps) : cut + 0.5f * whole;
    float rounds = fmaxf(1.f, groups * c.share);
    if (parts > 0.f) rounds = ceilf(rounds);
    float cost = fmaxf(rounds * (steps * c.step_cost + kFilling), work * heads * c.read_cost);
    if (lane > 0) cost += kJoining + groups * c.sums_cost;
    if (lane > 0 && (steps < kTreeSteps || most > c.slots)) cost = INFINITY;
    // The lane of the least cost; costs are positive, so their bits are in their order.
    const int least = 0x7f800000 - most_of_lanes(0x7f800000 - __builtin_bit_cast(int, cost));
    const int best = __builtin_ctzll(__ballot(__builtin_bit_cast(int, cost) == least) | (uint64_t(1) << 63));
    // Float32 steps may be one short of kMostParts parts where there are more than 2^23.
    return best == 0 ? longest : max(__builtin_amdgcn_readlane(static_cast<int>(steps), best), (longest + kMostParts - 1) / kMostParts);
}

// A tree's workgroup: of which sequence, tile of rows, K/V head and part of the keys.
//
// Of at most 64 sequences every wave looks at them all, a lane each, and the longest come
// first. Of more a kernel before this one says where each one's workgroups begin (1,024
// sequences of a token over 200 keys 283 us, by every workgroup itself 454). Within a sequence
// part, tile of rows, head: with eight heads (or 16, ..) the tiles of rows that share keys
// are on one XCD.
template <int kRows>
__device__ __forceinline__ bool tree_unit(const WindowCall& c, int id, WindowUnit& u) {
    const int lane = threadIdx.x & 63, group = static_cast<int>(c.group.d), heads = c.kv_heads;
    const int mine = id / heads;
    TreeSequence s;
    int each, start = 0;
    auto parts_of = [&](int steps) { return (steps + each - 1) / each; };
    if (c.starts) {
        each = c.starts[c.batch + 1];
        if (mine >= c.starts[c.batch]) return false;
        // The last sequence that begins at `mine` or before, a 64th of the range at a time.
        int first = 0;
        for (int range = c.batch; range > 1;) {
            const int step = (range + 63) / 64, at = lane * step;
            const int places = max(__popcll(__ballot(at < range && c.starts[min(first + at, c.batch)] <= mine)), 1) - 1;
            first += places * step;
            range = min(step, range - places * step);
        }
        u.b = __builtin_amdgcn_readfirstlane(first);
        s = tree_sequence<kRows>(c, u.b);
        start = c.starts[u.b];
    } else {
        s = tree_sequence<kRows>(c, lane);
        const int longest = most_of_lanes(s.steps);
        if (longest == 0) return false;
        const float its_tiles = static_cast<float>(s.tiles), its_steps = static_cast<float>(s.steps);
        const float work = lane_value(running_sum(its_tiles * its_steps, lane), 63);
        float parts = 0.f;
        const int units = lane_value(running_sum(s.tiles, lane), 63);
        // Counting takes 0.1 us a sequence, and gives nothing where whole tiles fill two rounds.
        if (kRows == 256 && work * heads * c.read_cost > 2.f * c.batch && static_cast<float>(units) * heads * c.share < 2.f) {
            const float one_by = 1.f / tree_steps(longest);
            for (int j = 0; j < c.batch; ++j) parts += lane_value(its_tiles, j) * ceilf(lane_value(its_steps, j) * one_by - 1e-5f);
        }
        each = tree_part(c, work, units, longest, parts);
        // In the order of the keys; there are at most 2^25 steps.
        const uint32_t key = static_cast<uint32_t>(s.steps) * 64 + 63 - lane;
        const int all = s.tiles * parts_of(s.steps);
        for (int j0 = 0; j0 < c.batch; j0 += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t other = __builtin_amdgcn_readlane(key, j0 + j);
                const int its = __builtin_amdgcn_readlane(all, j0 + j);
                start += other > key ? its : 0;
            }
        const uint64_t here = __ballot(mine >= start && mine < start + all);
        if (!here) return false;
        u.b = __builtin_ctzll(here);
        for (int* x : {&s.off, &s.n, &s.length, &s.tiles, &s.steps, &start}) *x = __builtin_amdgcn_readlane(*x, u.b);
    }
    for (int* x : {&each, &s.off, &s.n, &s.length, &s.tiles, &s.steps, &start}) *x = __builtin_amdgcn_readfirstlane(*x);
    u.parts = parts_of(s.steps);
    const int place = mine - start;
    // Offsets that do not ascend may give a sequence more tiles than were counted.
    if (place < 0 || place >= s.tiles * u.parts || (u.parts > 1 && id >= c.slots)) return false;
    u.part = __builtin_amdgcn_readfirstlane(place / s.tiles);
    u.tile = __builtin_amdgcn_readfirstlane(place - u.part * s.tiles);
    u.kv_head = __builtin_amdgcn_readfirstlane(id - mine * heads);
    u.stride = s.tiles * heads;
    u.slot = __builtin_amdgcn_readfirstlane(id);
    u.head = u.kv_head * group;
    u.off = s.off;
    u.n = s.n;
    u.length = s.length;
    u.first = u.length - u.n;
    return true;
}

constexpr int kPlanThreads = 1024;

// Of more than 64 sequences: the first workgroup of each (over all heads), how many
// there are, and the steps of a part. One workgroup, a thread for each sequence.
template <int kRows>
__global__ __launch_bounds__(kPlanThreads) void tree_plan_kernel(WindowCall c) {
    constexpr int kWaves = kPlanThreads / 64;
    __shared__ float works[kWaves];
    __shared__ int counts[kWaves], longests[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float work = 0.f;
    int units = 0, longest = 0;
    for (int b = tid; b < c.batch; b += kPlanThreads) {
        const TreeSequence s = tree_sequence<kRows>(c, b);
        work += static_cast<float>(s.tiles) * static_cast<float>(s.steps);
        units += s.tiles;
        longest = max(longest, s.steps);
    }
    works[wave] = lane_value(running_sum(work, lane), 63);
    counts[wave] = lane_value(running_sum(units, lane), 63);
    longests[wave] = most_of_lanes(longest);
    __syncthreads();
    work = 0.f, units = 0, longest = 1;
    for (int w = 0; w < kWaves; ++w) {
        work += works[w];
        units += counts[w];
        longest = max(longest, longests[w]);
    }
    const int each = tree_part(c, work, units, longest, 0.f);
    int before = 0;
    for (int b0 = 0; b0 < c.batch; b0 += kPlanThreads) {
        const TreeSequence s = tree_sequence<kRows>(c, b0 + tid);
        const int all = s.tiles * ((s.steps + each - 1) / each), sum = running_sum(all, lane);
        __syncthreads();
        counts[wave] = lane_value(sum, 63);
        __syncthreads();
        for (int w = 0; w < wave; ++w) before += counts[w];
        if (b0 + tid < c.batch) c.starts[b0 + tid] = before + sum - all;
        for (int w = wave; w < kWaves; ++w) before += counts[w];
    }
    if (tid == 0) {
        c.starts[c.batch] = before;
        c.starts[c.batch + 1] = each;
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
    static constexpr int kMasks = kVotes + 32;  // a tree's masks, behind the others
};

// Words of a tree's masks: what fits two workgroups of four waves to a CU, or one of eight.
template <int kWaves>
constexpr int kMaskWords = kWaves == 4 ? 3968 : 16384;

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

// Of a word of a line, whose tokens' depths go up to `depth` (moved to the next word's),
// those of at least `from` or below `sinks`.
__device__ __forceinline__ uint64_t within(uint64_t word, int& depth, int from, int sinks) {
    const int count = __popcll(word), first = depth - count + 1;
    depth = first - 1;
    uint64_t late = word, rest = word;
    for (int i = min(from - first, count); i > 0; --i) late &= late - 1;
    for (int i = min(sinks - first, count); i > 0; --i) rest &= rest - 1;
    return late | (word & ~rest);
}

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

extern __shared__ __align__(16) unsigned char smem[];

template <class T, int D, bool kPaged, bool kSplit, bool kTree, int kWaves = 4>
__device__ __forceinline__ void window_rows(const WindowCall& c, const WindowUnit& u) {
    using Tile = WindowTile<T, D>;
    constexpr int kSteps = Tile::kSteps, kBlocks = Tile::kBlocks, kOps = Tile::kOps;
    constexpr int kRows = 32 * kWaves, kThreads = 64 * kWaves;
    // Of eight waves four transfer K and four V.
    constexpr bool kApart = kWaves == 8;
    static_assert(kWaves == 4 || (kApart && kTree));
    const bool split = kSplit && (!kTree || u.parts > 1);
    const int group = kPaged ? c.group.d : 1;
    int tid = threadIdx.x;
    if constexpr (kTree) asm volatile("" : "+v"(tid));  // not known from tree_unit, whose values would be kept for it
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int loader = kApart ? wave & 3 : wave;  // transfers keys 8 loader .. + 7 of a tile

    // Bounds of the rows r0 .. r1 of the tile that exist: keys that some row
    // sees, and those that every row sees.
    const WindowMask mask = c.mask;
    const int row0 = u.tile * kRows, rows = min(kRows, u.n * group - row0);
    auto token_at = [&](int r) { return kPaged ? (row0 + r) / group : row0 + r; };
    // A tree's tokens are at positions from u.first on, and see nothing in the cache behind their own place.
    const int p_first = max(u.first + (kTree ? 0 : token_at(0)), 0), p_last = min(u.first + token_at(rows - 1), u.length - 1);
    TileRange range;
    range.set(mask, p_first, p_last, u.length);
    const int end = range.end;
    int tile0 = 0, tiles = range.tiles;
    if constexpr (kSplit) {
        const int part = kTree ? u.part : blockIdx.y, parts = kTree ? u.parts : c.parts;
        tile0 = static_cast<int>(int64_t(tiles) * part / parts);
        tiles = static_cast<int>(int64_t(tiles) * (part + 1) / parts) - tile0;
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
    int masks[2];                  // of a tree instead: where the masks of the row's token are in LDS
    if constexpr (!kTree) {
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
    }
    // Tiles that every row of this wave (of a tree: of the workgroup) sees need no mask: keys
    // from full_low to full_high, and those before full_sink. A wave with a row that exists
    // but sees nothing masks every tile.
    int full_low = 0, full_high = 0, full_sink = 0;
    const int wave_rows = min(32, rows - wave * 32);
    const bool active = wave_rows > 0;
    if (kTree || active) {
        const int pf = u.first + (kTree ? 0 : token_at(wave * 32)), pl = u.first + token_at(kTree ? rows - 1 : wave * 32 + wave_rows - 1);
        if (pf >= 0 && pl < u.length) {
            full_low = mask.low(pl);
            full_high = kTree ? pf : mask.high(pf, u.length);
            full_sink = min(mask.sinks, full_high);
        }
    }

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)smem));
    const char* kbase = static_cast<const char*>(c.k) + ((kPaged ? 0 : u.b * c.k_rows.batch) + u.kv_head * c.k_rows.head) * 2;
    const char* vbase = static_cast<const char*>(c.v) + ((kPaged ? 0 : u.b * c.v_rows.batch) + u.kv_head * c.v_rows.head) * 2;
    const uint32_t k_token = static_cast<uint32_t>(c.k_rows.token * 2), v_token = static_cast<uint32_t>(c.v_rows.token * 2);
    const int32_t* table = kPaged ? c.table + int64_t(u.b) * c.table_width : nullptr;
    const int last_entry = c.table_width - 1;

    // What a tree's masks are made of is asked for beside the page table, and read again later.
    int token_position = 0, token_above = 0;
    uint64_t token_near = 0;
    if constexpr (kTree) {
        const int token = u.off + token_at(min(tid & (kRows - 1), rows - 1));
        token_position = c.positions[token];
        token_above = c.above[token];
        token_near = c.near[token];
    }

    // Whether a key that some row would see lies on no page (then every tile
    // asks the table for its keys). Pages between the sinks and the window, which
    // may have been given back, do not count.
    bool holes = false;
    auto any_vote = [&](const uint32_t* votes) {
        u32x4 all = *reinterpret_cast<const u32x4*>(votes);
        if constexpr (kWaves == 8) all |= *reinterpret_cast<const u32x4*>(votes + 4);
        return __builtin_amdgcn_readfirstlane(all[0] | all[1] | all[2] | all[3]) != 0;
    };
    if constexpr (kPaged) {
        bool bad = false;
        auto scan = [&](int from, int to) {
            const int page = static_cast<int>(c.page.d);
            for (int i = from / page + tid; from < to && i <= (to - 1) / page; i += kThreads)
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
        holes = any_vote(votes);
    }
    if constexpr (kTree) asm volatile("" ::"v"(token_position), "v"(token_above), "v"(token_near));
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
        const int key = lane / kChunks, pos = lane % kChunks, in_tile = 8 * loader + Tile::kOpKeys * e + key;
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
            const uint32_t key = next_key + 8 * loader;
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
        const int key = next_key + 8 * loader;
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
            buffer_to_lds(buffer, src[0] + at, src[1] + at, lds + loader * (8 * D * 2));
        else
            buffer_to_lds(buffer, src[0] + at, lds + loader * (8 * D * 2));
    };
    auto move_k = [&](int t, const Place& p) {
        if (kApart && wave >= 4) return;
        move(kbase, c.k_rows, k_token, k_less, k_all, k_src, p, lds0 + (t & (kRing - 1)) * Tile::kBytes);
    };
    auto move_v = [&](int t, const Place& p) {
        if (kApart && wave < 4) return;
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
    // Of a masked tile of a tree: which one it is.
    auto mask_of = [&](int t) { return t - clear_sink - (t >= clear_from ? clear : 0); };
    // Bit r of the result: key 16h + 4lg + r of tile t is seen by row 16j + li.
    auto seen_keys = [&](int t, int h, int j) {
        if constexpr (kTree) {
            if (t >= tiles) return 0u;
            if (!is_masked(t)) return 15u;
            const uint32_t* its = reinterpret_cast<const uint32_t*>(smem + Tile::kMasks) + masks[j];
            return its[mask_of(t)] >> (16 * h + 4 * lg) & 15u;
        } else {
            const int key = range.key(tile0 + t) + 16 * h + 4 * lg;
            uint32_t bits = 0;
            if (t < tiles && (!kPaged || !holes || on_page(key)))
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    bits |= static_cast<uint32_t>(key + r - low[j]) < static_cast<uint32_t>(seen[j]) || key + r < sink[j] ? 1u << r : 0u;
            return bits;
        }
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
    bool first_pass = true;
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
            landed_and_barrier<(kApart ? 2 : 4) * kOps>();
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
            Place p0, p1, p2;
            if constexpr (kTree) {
                // The page table's entries of six tiles at once, a lane each.
                const uint32_t key = range.key(tile0 + min(lane, 5)) + 8 * loader, near = __umulhi(key, c.page.m), rest = key - near * c.page.d;
                const bool more = rest >= c.page.d;
                const int entry = table[min(more ? near + 1 : near, static_cast<uint32_t>(last_entry))], at = more ? rest - c.page.d : rest;
                auto place = [&](int t) {
                    next_entry = __builtin_amdgcn_readlane(entry, t);
                    next_at = __builtin_amdgcn_readlane(at, t);
                    return next_place();
                };
                p0 = place(0);
                p1 = place(1);
                p2 = place(2);
                vp = place(3);
                mp = place(4);
                kp = place(5);
            } else {
                p0 = ask_place();
                p1 = ask_place();
                p2 = ask_place();
                vp = ask_place();
            }
            move_k(0, p0);
            move_k(1, p1);
            move_k(2, p2);
            move_v(0, p0);
            move_k(3, vp);
            move_v(1, p1);
            move_v(2, p2);
        }
        if (!kTree || first_pass) {
            if (active) read_q();  // behind the transfers, not before them
        }
        if constexpr (!kTree) {
            mp = ask_place();
            kp = ask_place();
        }
        f32x4 s0[4], s1[4];
        u32x4 ka[2 * kSteps];
        float mx[2] = {-INFINITY, -INFINITY};
        landed_and_barrier<(kApart ? 2 : 5) * kOps>();
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
                    s0[n][r] = kTree ? __builtin_fmaf(s0[n][r], c.scale_log2, -m_run[n & 1]) : s0[n][r] * c.scale_log2;
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
        return any_vote(votes);
    };

    // The same sums, tile by tile, with values that are not finite kept from the
    // rows that do not see them: V without them, and where a row sees one, an
    // infinity of its sign (or, for NaN, of both).
    auto careful_pass = [&]() {
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
    if constexpr (kTree) {
        // A tree's masks lie in LDS: for each of the tile's tokens a word for each masked tile of
        // keys. Where they do not all fit (128 tokens and more than 31 masked tiles, or 256
        // and 64) the tiles are taken in segments. (Made behind the first transfers they cost
        // the same: 8 ragged sequences 37 us, this way 36.)
        const int base = u.first, token0 = token_at(0), tokens = token_at(rows - 1) - token0 + 1, fit = kMaskWords<kWaves> / tokens;
        const int part0 = tile0, part_tiles = tiles;
        // In tiles of the part: clear ones are 0 .. sinks_end - 1 and window .. window_end - 1.
        const int sinks_end = max(clear_sink, 0), window = max(clear_from, sinks_end), window_end = max(clear_from + clear, window);
        const bool cut = mask.low(max(p_last, 0)) > base;
        // What p sees of the cached keys from key0 on.
        auto cached = [&](int p, int low_of, int key0) {
            auto below = [&](int key) {  // keys of the tile before it
                const int n = min(max(key - key0, 0), kWindowKeys);
                return n == kWindowKeys ? ~0u : (1u << n) - 1;
            };
            return p < 0 ? 0u : (below(base) & ~below(low_of)) | below(min(mask.sinks, max(base, 0)));
        };
        auto paged = [&](int key0) {
            uint32_t bits = ~0u;
            if (holes)
                for (int g = 0; g < 4; ++g)
                    if (!on_page(key0 + 8 * g)) bits &= ~(0xffu << (8 * g));
            return bits;
        };
        auto each_segment = [&](auto pass) {
            bool odd = false;
            for (int from = 0, to = 0; from < part_tiles; from = to) {
                // As many tiles as have `fit` masked ones.
                int left = fit, at = max(from, sinks_end);
                if (at < window) {
                    const int run = min(window - at, left);
                    left -= run;
                    at += run;
                }
                if (at >= window) at = max(at, window_end) + left;
                to = min(part_tiles, at);
                tile0 = part0 + from;
                tiles = to - from;
                clear_sink = max(sinks_end - from, 0);
                clear_from = max(window - from, clear_sink);
                clear = max(window_end - from - clear_from, 0);
                const int masked = max(0, min(tiles, clear_from) - clear_sink) + max(0, tiles - clear_from - clear);
                auto tile_of = [&](int w) { return w + clear_sink + (w + clear_sink >= clear_from ? clear : 0); };
                uint32_t* words = reinterpret_cast<uint32_t*>(smem + Tile::kMasks);
                // The last `drafts` of the masked tiles have drafts among their keys.
                int drafts = 0;
                while (drafts < masked && range.key(tile0 + tile_of(masked - 1 - drafts)) + kWindowKeys > base) ++drafts;
                int thread = tid;
                asm volatile("" : "+v"(thread));  // nothing made of it is kept in registers beside the passes
                for (int t = thread & (kRows - 1); t < tokens; t += kRows) {
                    int i = token0 + t;  // the last token of its line that has not been looked at
                    const int p = c.positions[u.off + i];
                    int up = c.above[u.off + i];
                    uint64_t its = c.near[u.off + i];
                    const int low_of = mask.low(max(p, 0));
                    for (int w = thread / kRows; w < masked - drafts; w += kThreads / kRows) {
                        const int key0 = range.key(tile0 + tile_of(w));
                        words[t * masked + w] = cached(p, low_of, key0) & paged(key0);
                    }
                    if (thread >= kRows || drafts == 0) continue;
                    // Up the token's line, in words of 64 places, as the tiles of drafts go down.
                    int depth = p - base, block = -1;
                    uint64_t word = 0;
                    auto half = [&](int h) {  // places 32h .. 32h + 31
                        if (h < 0) return 0u;
                        if (h >> 1 != block) {
                            block = h >> 1;
                            word = 0;
                            while (i >= 64 * block && i >= 0) {
                                const int place = i & ~63;
                                if (cut) its = within(its, depth, low_of - base, mask.sinks - base);
                                if (place == 64 * block) word = its;
                                i = up < place ? up : -1;
                                if (i >= 0) {
                                    its = c.near[u.off + i];
                                    up = c.above[u.off + i];
                                }
                            }
                        }
                        return static_cast<uint32_t>(word >> (32 * (h & 1)));
                    };
                    uint32_t upper = 0;
                    for (int w = masked - 1; w >= masked - drafts; --w) {
                        const int key0 = range.key(tile0 + tile_of(w)), place = key0 - base;
                        if (w == masked - 1) upper = half((place >> 5) + 1);
                        const uint32_t lower = half(place >> 5);
                        const uint32_t line = __builtin_amdgcn_alignbit(upper, lower, place & 31);
                        upper = lower;
                        words[t * masked + w] = (cached(p, low_of, key0) | (p < 0 ? 0u : line)) & paged(key0);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = row0 + min((thread >> 6) * 32 + 16 * j + (thread & 15), rows - 1);
                    masks[j] = (row / group - token0) * masked;
                }
                odd |= pass();
                first_pass = false;
            }
            return odd;
        };
        if (each_segment(fast_pass)) {
            reset();
            each_segment([&]() {
                careful_pass();
                return false;
            });
        }
    } else if (tiles > 0 && fast_pass()) {
        reset();
        careful_pass();
    }

    if (!active) return;
    const WindowCall& e = kTree ? arguments() : c;  // the rest of the call
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
        const int64_t stat_at = u.b * e.row.batch + head * e.row.head + int64_t(u.off + token) * e.row.token;
        const int place = wave * 32 + 16 * j + li;
        if (kTree && u.part == 0 && lg == 0) e.row_parts[stat_at] = make_int4(u.slot, u.parts, place, u.stride);
        if (split) {
            const int64_t at = kTree ? int64_t(u.slot) * kRows + place : blockIdx.y * e.rows + stat_at;
            if (lg == 0) {
                e.partial_stat[at] = float2{slack[j] == kSlack<T> ? m_run[j] : -INFINITY, l};
                if (!kPaged && e.out_rest) e.partial_rounded[at] = rounded;
            }
            if (l == 0.f) continue;
            float* dst = e.partial_o + at * D + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4*>(dst + 16 * b) = o_acc[b][j];
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l, better = kPaged || rounded == 0.f ? inv : 1.0f / rounded;
            uint16_t* orow = static_cast<uint16_t*>(e.out) + u.b * e.out_rows.batch + head * e.out_rows.head +
                             int64_t(u.off + token) * e.out_rows.token + 4 * lg;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const f32x4 o = o_acc[b][j] * inv;
                const u32x2 w = {T::pack(o[0], o[1]), T::pack(o[2], o[3])};
                *reinterpret_cast<u32x2*>(orow + 16 * b) = w;
                if (!kTree && e.out_rest) {
                    const f32x4 before = o_acc[b][j] * better;
                    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(e.out_rest) + (orow - static_cast<uint16_t*>(e.out)) + 16 * b) =
                        u32x2{rest_of<T>(before[0], before[1], w[0]), rest_of<T>(before[2], before[3], w[1])};
                }
            }
            if (e.lse && lg == 0) e.lse[stat_at] = l == 0.f ? -INFINITY : m_run[j] + log2f(l);
        }
    }
}

template <class T, int D, bool kPaged, bool kSplit>
__global__ __launch_bounds__(kWindowThreads, 2) void window_kernel(WindowCall c, WindowGrid places) {
    touch(c.q, c.k_rows.batch, c.row.batch, c.lengths, c.rows, places.heads);
    WindowUnit u;
    if (window_unit<kPaged>(c, places, blockIdx.x, u)) window_rows<T, D, kPaged, kSplit, false>(c, u);
}

template <class T, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, D == 64 && kWaves == 4 ? 3 : 2) void tree_attention_kernel(WindowCall c) {
    touch(c.q, c.k_rows.batch, c.row.batch, c.lengths, c.rows, c.near);
    WindowUnit u;
    if (tree_unit<32 * kWaves>(arguments(), blockIdx.x, u)) window_rows<T, D, true, true, true, kWaves>(arguments(), u);
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

// A tree's split rows, as above: 16 lanes take a row of a part. Few rows: the four groups of
// a wave take every fourth part of one row; many: a row each. Statistics and values are
// asked for together, four parts ahead, so a row takes two loads after one another (the
// first says where the parts are) for up to four parts of a group.
template <class T, int D, int kGroups>
__global__ __launch_bounds__(256) void tree_combine_kernel(WindowCall c) {
    const int lane = threadIdx.x & 63, of16 = lane & 15, group = kGroups == 4 ? lane >> 4 : 0;
    const int64_t row = int64_t(blockIdx.x) * (16 / kGroups) + (kGroups == 4 ? threadIdx.x >> 6 : threadIdx.x >> 4);
    if (row >= c.rows) return;
    const int token = static_cast<int>(static_cast<uint32_t>(row / c.heads)), head = static_cast<int>(row - int64_t(token) * c.heads);
    const int4 its = c.row_parts[row];
    // Rows before the first sequence and behind the last stay as they were.
    if (token < c.offsets[0] || token >= c.offsets[c.batch]) return;
    const int parts = its.y, slot = its.x, in_tile = its.z;
    // One part has been written whole; a row that offsets which do not ascend leave out may
    // hold anything.
    if (parts < 2 || parts > kMostParts || slot < 0 || its.w < 0 || in_tile < 0 || in_tile >= c.tile_rows ||
        slot + int64_t(its.w) * (parts - 1) >= c.slots)
        return;
    auto place = [&](int p) { return (slot + int64_t(its.w) * p) * c.tile_rows + in_tile; };
    // An infinite value is seen however small its part's weight is.
    auto weighted = [](float w, float x) { return w == 0.f && !(fabsf(x) < INFINITY) ? x : w * x; };
    constexpr int kEach = D / 16, kAhead = 4;
    float m = -INFINITY, l = 0.f, o[kEach] = {};
    for (int p0 = 0; p0 < parts; p0 += kGroups * kAhead) {
        float2 stat[kAhead];
        f32x4 x[kAhead][kEach / 4];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int p = p0 + kGroups * i + group;
            stat[i] = float2{-INFINITY, 0.f};
#pragma unroll
            for (int e = 0; e < kEach / 4; ++e) x[i][e] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (p < parts) {
                const int64_t at = place(p);
                stat[i] = c.partial_stat[at];
#pragma unroll
                for (int e = 0; e < kEach / 4; ++e) x[i][e] = *reinterpret_cast<const f32x4*>(c.partial_o + at * D + of16 * kEach + 4 * e);
            }
        }
        float top = m;  // a part without a key has written no row
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (stat[i].y != 0.f) top = fmaxf(top, stat[i].x);
        const float before = l == 0.f ? 0.f : fast_exp2(m - top);
        l *= before;
#pragma unroll
        for (int e = 0; e < kEach; ++e) o[e] = weighted(before, o[e]);
        m = top;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (stat[i].y == 0.f) continue;
            const float w = fast_exp2(stat[i].x - m);
            l += w * stat[i].y;
#pragma unroll
            for (int e = 0; e < kEach; ++e) o[e] += weighted(w, x[i][e / 4][e % 4]);
        }
    }
    // The groups.
#pragma unroll
    for (int s = 16; s < 16 * kGroups; s *= 2) {
        const float its_m = __shfl_xor(m, s), its_l = __shfl_xor(l, s), top = fmaxf(m, its_m);
        const float w = l == 0.f ? 0.f : fast_exp2(m - top), its_w = its_l == 0.f ? 0.f : fast_exp2(its_m - top);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const float mine = weighted(w, o[e]), its = weighted(its_w, __shfl_xor(o[e], s));
            o[e] = mine + its;
        }
        l = w * l + its_w * its_l;
        m = top;
    }
    if (group != 0) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint16_t* out = static_cast<uint16_t*>(c.out) + head * c.out_rows.head + int64_t(token) * c.out_rows.token + of16 * kEach;
#pragma unroll
    for (int e = 0; e < kEach; e += 4)
        *reinterpret_cast<u32x2*>(out + e) = u32x2{T::pack(o[e] * inv, o[e + 1] * inv), T::pack(o[e + 2] * inv, o[e + 3] * inv)};
    if (c.lse && of16 == 0) c.lse[row] = l == 0.f ? -INFINITY : m + log2f(l);
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

// Rows of partial results that are added up by a wave each: fewer than fill the chip with
// four rows to a wave (512 rows of 32 parts: 9.6 us, a wave and four loads at a time 15.3;
// 19,000 rows of 2 or 3 parts, four to a wave 8.4 us, a wave each 18).
constexpr int64_t kFewRows = 4096;

template <class T, int D, int kWaves>
int launch_tree_as(const WindowCall& c, hipStream_t stream) {
    const auto kernel = tree_attention_kernel<T, D, kWaves>;
    constexpr int kLds = WindowTile<T, D>::kMasks + 4 * kMaskWords<kWaves>;
    if (int rc = ensure_lds_limit(reinterpret_cast<const void*>(kernel), kLds)) return rc;
    if (c.starts) {
        hipLaunchKernelGGL(tree_plan_kernel<32 * kWaves>, dim3(1), dim3(kPlanThreads), 0, stream, c);
        if (int rc = check_launch("tree_plan_kernel")) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(c.groups)), dim3(64 * kWaves), kLds, stream, c);
    if (int rc = check_launch("tree_attention_kernel")) return rc;
    if (c.rows <= kFewRows)
        hipLaunchKernelGGL((tree_combine_kernel<T, D, 4>), dim3(static_cast<unsigned>((c.rows + 3) / 4)), dim3(256), 0, stream, c);
    else
        hipLaunchKernelGGL((tree_combine_kernel<T, D, 1>), dim3(static_cast<unsigned>((c.rows + 15) / 16)), dim3(256), 0, stream, c);
    return check_launch("tree_combine_kernel");
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

// The parts themselves are tree_unit's, which keeps to the groups and slots given here.
//
// Tiles of 256 rows, for eight waves, where sequences have more than 128 rows on average: keys
// are then read once for twice the rows (one sequence of 64 drafts, 256 rows of 100,000
// keys, with the joining of parts: 136 us, in tiles of 128 rows 193). Not with D = 64, whose
// four waves take a third of a CU (4 x 701 drafts 82 us, of eight waves a quarter more).
void plan_tree(WindowCall& c, int64_t most_keys) {
    const int64_t packed = int64_t(c.tokens) * c.group.d;
    c.tile_rows = c.dim == 128 && packed > int64_t(c.batch) * 128 ? 256 : 128;
    // A sequence of x rows has at most (x - 1) / tile_rows + 1 tiles of rows.
    const int64_t units = (packed <= c.batch ? packed : (packed - c.batch) / c.tile_rows + c.batch) * c.kv_heads;
    const int64_t steps = (most_keys + 2 * kWindowKeys - 1) / kWindowKeys + 1;
    const int64_t parts = std::min<int64_t>(kMostParts, (steps + kTreeSteps - 1) / kTreeSteps);
    const int64_t at_once = c.tile_rows == 256 ? 256 : c.dim == 128 ? 512 : 768;
    c.slots = static_cast<int32_t>(std::min(units * parts, 2 * at_once));
    c.groups = static_cast<int32_t>(std::max<int64_t>(units, c.slots));
    c.share = 1.f / float(at_once);
    c.step_cost = c.tile_rows == 256 ? 1.1f : c.dim == 128 ? 0.9f : 0.55f;
    c.read_cost = float(kWindowKeys * c.dim * 4) / 4.7e6f;
    const double rows = std::min<double>(c.tile_rows, double(packed) / c.batch);
    c.sums_cost = static_cast<float>(rows * (c.dim * 4.0 + 8) * 2 / 4.5e6);
}

int launch_window(const WindowCall& c, hipStream_t stream) {
    auto typed = [&](auto t) {
        using T = decltype(t);
        if (c.near)
            return c.dim == 64 ? launch_tree_as<T, 64, 4>(c, stream)
                               : c.tile_rows == 128 ? launch_tree_as<T, 128, 4>(c, stream) : launch_tree_as<T, 128, 8>(c, stream);
        if (c.dim == 128) return c.paged ? launch_as<T, 128, true>(c, stream) : launch_as<T, 128, false>(c, stream);
        return c.paged ? launch_as<T, 64, true>(c, stream) : launch_as<T, 64, false>(c, stream);
    };
    return c.half ? typed(F16{}) : typed(Bf16{});
}

}  // namespace ab
