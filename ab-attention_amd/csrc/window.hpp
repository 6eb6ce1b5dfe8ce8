// Windowed causal attention: the mask, the element types and the LDS tiles that
// its forward and backward kernels share.
#pragma once

#include "common.hpp"
#include "layout.hpp"

namespace ab {

// The mask. Tokens are grouped into frames of `frame` tokens (1: plain causal
// attention). The query at position p sees the keys of its own frame and of
// earlier ones down to `back` tokens before its frame's first, and the first
// `sinks` tokens, as far as they are not later than its frame:
//   [0, min(sinks, high)) and [low, high),  low = max(0, start - back),
//   high = min(start + frame, length),      start = p - p % frame.
// All three bounds grow with p. Positions, back, sinks and frame are at most
// 2^30, so the sums stay inside 32 bits.
struct WindowMask {
    Divisor frame;
    int32_t back, sinks;
    __device__ __forceinline__ int start(int p) const {
        uint32_t q = __umulhi(static_cast<uint32_t>(p), frame.m);
        uint32_t rest = static_cast<uint32_t>(p) - q * frame.d;
        if (rest >= frame.d) rest -= frame.d;
        return p - static_cast<int>(rest);
    }
    __device__ __forceinline__ int low(int p) const { return max(0, start(p) - back); }
    __device__ __forceinline__ int high(int p, int length) const {
        return min(start(p) + static_cast<int>(frame.d), length);
    }
};

// The bf16 and fp16 forms of what the kernels do with 16-bit elements.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) unsigned char lds_u8;

struct Bf16 {
    // D = A B + C of 16x16x32 (A: 16 x 32, lane l row l % 16, k 8(l / 16) .. + 7;
    // B: 32 x 16, lane l column l % 16, the same k; C and D: lane l column
    // l % 16, rows 4(l / 16) .. + 3).
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
    // c + both halves.
    static __device__ __forceinline__ float add(uint32_t w, float c) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, kOne * 0x10001u), c, false);
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
    // Exponent bits of both halves, and what turns an exponent of all ones into
    // the half's sign bit when added.
    static constexpr uint32_t kExponent = 0x7f807f80u, kOverflow = 0x00800080u, kOne = 0x3f80u;
    static constexpr int kLift = 0;  // log2 of what probabilities are rounded as multiples of
};

struct F16 {
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    }
    static __device__ __forceinline__ float add(uint32_t w, float c) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, kOne * 0x10001u), c, false);
    }
    static __device__ __forceinline__ float lo(uint32_t w) {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
    }
    static __device__ __forceinline__ float hi(uint32_t w) {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
    }
    static constexpr uint32_t kExponent = 0x7c007c00u, kOverflow = 0x04000400u, kOne = 0x3c00u;
    static constexpr int kLift = 10;
};

// Transposing LDS read: within each 16-lane group, lane i receives element
// i % 4 of the 8 bytes read by lanes 4r + i / 4, for r = 0..3.
__device__ __forceinline__ i16x4 lds_read_transposed(uint32_t lds) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(static_cast<uintptr_t>(lds)));
}

__device__ __forceinline__ u32x4 lds_read16(uint32_t lds) {
    return *reinterpret_cast<const lds_u32x4*>(static_cast<uintptr_t>(lds));
}

// A buffer of `bytes` bytes from `base` on, the same in all lanes: reads past its
// end give zeros.
__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes per lane from the buffer, at an offset of its own in each lane,
// straight into LDS: lane j writes bytes [lds + 16j, lds + 16j + 16); a lane
// past the buffer's end writes zeros. Counted by vmcnt. The wait states are
// those between scalar writes of m0 or the descriptor and their use.
__device__ __forceinline__ void buffer_to_lds(u32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer)
                 : "memory", "m0");
}
// The same twice, into 1 KiB each.
__device__ __forceinline__ void buffer_to_lds(u32x4 buffer, uint32_t offset0, uint32_t offset1, uint32_t lds) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "s_add_u32 m0, %0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" ::"s"(lds),
        "v"(offset0), "v"(offset1), "s"(buffer)
        : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

// The first thing each of these kernels does: a value from every 64-byte line of
// its arguments (in host memory) at once, so that the lines arrive together and not
// one after the other where the compiler first needs them.
template <class A, class B, class C, class D, class E, class F>
__device__ __forceinline__ void touch(A a, B b, C c, D d, E e, F f) {
    asm volatile("" ::"s"(a), "s"(b), "s"(c), "s"(d), "s"(e), "s"(f));
}

// At most N of this wave's vector memory operations still in flight, none of
// its LDS ones; then a workgroup barrier that the compiler moves no memory
// access across.
template <int N>
__device__ __forceinline__ void landed_and_barrier() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
    asm volatile("s_barrier" ::: "memory");
}

// A tensor of rows of `dim` 16-bit elements; strides in elements.
struct Rows {
    int64_t batch, head, token;
};

// One call of the forward pass. Rows of Q are read at q + b q.batch + h q.head +
// t q.token; `paged`, over a cache, K and V at k.batch * page + h k.head +
// (token in the page) k.token, and batch item b's queries are the packed rows
// offsets[b] .. offsets[b + 1]. `row` gives the place of a query's normaliser.
struct WindowCall {
    const void *q, *k, *v;
    void *out, *out_rest;  // out_rest: what out lacks of a better one, or none
    float* lse;
    Rows q_rows, k_rows, v_rows, out_rows, row;
    int32_t batch, heads, kv_heads, tokens;  // tokens: of a batch item, or packed rows in all
    int32_t dim, half;                       // half: 0 bf16, 1 fp16
    bool paged;
    const int32_t *lengths, *offsets, *table;
    // New tokens that are a tree (TreeCall's results), or none.
    const int32_t *positions, *above;
    const uint64_t* near;
    int32_t table_width, pages;
    Divisor page, group;                     // tokens of a page; query heads of a K/V head
    WindowMask mask;
    float scale_log2;
    int32_t parts;                           // parts that every tile's keys are split into
    float* partial_o;                        // [parts][rows][dim] with workspace
    float2* partial_stat;                    // [parts][rows]: reference and sum
    float* partial_rounded;                  // [parts][rows], for a tensor's out_rest: sum of the rounded weights
    int64_t rows;                            // queries times heads
    // Of a tree, whose parts are chosen by the kernel: workgroups, places for parts' rows
    // [slots][tile_rows], rows of a tile; one by the workgroups that run at once; and in us what
    // a step costs, the reading of its keys, and writing and reading the sums of a part.
    int32_t groups, slots, tile_rows;
    float share, step_cost, read_cost, sums_cost;
    int4* row_parts;                         // [rows]: first place, parts, row in the place, from place to place
    int32_t* starts;                         // of more than 64 sequences [batch + 2]: tree_plan_kernel's
};

// One call of the backward pass over strided tensors. `stat` holds, for every
// 32 queries of a head, their 32 normalisers and 32 values of -delta.
struct WindowGradCall {
    const void *q, *k, *v, *out, *out_rest, *dout;  // out_rest: or none
    const float *lse, *dlse;  // dlse: of the normalisers, or none
    void *dq, *dk, *dv;
    Rows q_rows, k_rows, v_rows, out_rows, dout_rows, dq_rows, dk_rows, dv_rows;
    int32_t batch, heads, kv_heads, tokens, dim, half;
    const int32_t* lengths;
    int32_t group;
    WindowMask mask;
    float scale, scale_log2;
    float* stat;
    // Parts that the streamed rows of a tile are split into: of the first sink_tiles
    // key tiles, of the others, of query tiles.
    int32_t sink_tiles, sink_parts, key_parts, query_parts;
    // Their float32 sums: [heads][tiles][parts][dK, dV][128][dim] of the sinks' tiles,
    // then of the other key tiles, then [heads][tiles][parts][128][dim] of query tiles.
    float* partial;
};

constexpr int kWindowThreads = 256;
constexpr int kWindowRows = 128;  // query rows of a workgroup
constexpr int kTreeSteps = 4;     // tiles of keys of a part of a tree's, at least
constexpr int kMostParts = 64;    // of a tile of rows
constexpr float kFilling = 9.f;   // us that filling and emptying a workgroup's pipeline takes
constexpr float kJoining = 6.f;   // and the second kernel of parts
constexpr int kWindowKeys = 32;   // keys of a tile

// Keys of a run of tiles: the first `sink_tiles` tiles start at 0, the others at
// `window`; together they hold every key that some position from p_first to
// p_last sees, once.
struct TileRange {
    int sink_tiles, window, tiles, end;  // end: keys from here on are seen by none
    __device__ __forceinline__ int key(int u) const {
        return kWindowKeys * (u < sink_tiles ? u : u - sink_tiles) + (u < sink_tiles ? 0 : window);
    }
    __device__ __forceinline__ void set(const WindowMask& mask, int p_first, int p_last, int length) {
        sink_tiles = window = tiles = end = 0;
        if (p_last < p_first) return;
        const int low = mask.low(p_first);
        end = mask.high(p_last, length);
        const int sinks = min(mask.sinks, end);
        if (low > sinks) {
            sink_tiles = (sinks + kWindowKeys - 1) / kWindowKeys;
            window = max(low & ~7, sink_tiles * kWindowKeys);
        }
        tiles = sink_tiles + max(0, end - window + kWindowKeys - 1) / kWindowKeys;
    }
};

// Workgroup index -> (head, tile), without gaps: workgroups are dealt round-robin
// over the 8 XCDs in order, and one that has nothing to do keeps an XCD's place
// empty until the others' turn has come (40 heads x 37 tiles with three gaps in
// 40: 3,830 us instead of 3,285).
// The list: the last eight tiles (the longest) of every head, one for each XCD, then
// the eight before them, so that short rows end the call. Groups of 4 to 32
// neighbouring tiles for each XCD, whose windows overlap in its L2, fetch half as
// much but are slower nearly everywhere, for they do not start together (12 heads of
// 480p, window of 4 frames: 1,508 us, in groups 1,560 to 1,740; causal 16 x 16,384
// 1,112, in groups 1,139 to 1,707), and so are whole heads one after the other (1,640;
// 1,235).
struct WindowGrid {
    static constexpr uint32_t kRun = 8;
    uint32_t heads, tiles;
    unsigned size() const { return heads * tiles; }
    __device__ __forceinline__ void place(uint32_t n, int& head, int& tile) const {
        const uint32_t runs = tiles / kRun, whole = runs * kRun * heads;
        uint32_t each = kRun, first = 0;
        if (n < whole) {
            first = n / (kRun * heads);
            n -= first * kRun * heads;
            first *= kRun;
        } else {
            n -= whole;
            each = tiles - runs * kRun;
            first = runs * kRun;
        }
        head = n / each;
        tile = tiles - 1 - (first + n - head * each);
    }
};
inline WindowGrid window_grid(int64_t heads, int64_t tiles) { return {static_cast<uint32_t>(heads), static_cast<uint32_t>(tiles)}; }

int launch_window(const WindowCall& call, hipStream_t stream);
int window_parts(const WindowCall& call, int64_t most_keys);
int64_t window_tiles(const WindowCall& call);
// Sets what is said above of a tree's call.
void plan_tree(WindowCall& call, int64_t most_keys);
int launch_window_grad(const WindowGradCall& call, hipStream_t stream);
// Sets the tiles and parts of a split; returns the floats of stat and of partial.
void plan_window_grad(WindowGradCall& call, int64_t& stat, int64_t& partial);

}  // namespace ab
