// Windowed causal attention, backward.
//
// With P = 2^(S scale log2(e) - lse) recomputed from the forward pass'
// normalisers, S = Q K^T, and delta = rowsum(dO o O) - dlse / ln 2,
//   dV = P^T dO,  dS = P o (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q.
// Two kernels of one shape, so that every sum has one owner and one order (no
// atomics): a workgroup owns 128 rows, 32 a wave, kept in registers, and streams
// tiles of 32 rows of the other side through LDS:
//   queries: X = (Q, dO) owned, Y = (K, V) streamed, dQ += Y1^T dS,
//   keys:    X = (K, V) owned, Y = (Q, dO) streamed (of all query heads that
//            share them, one after the other), dK += Y1^T dS, dV += Y2^T P,
// each with S^T = Y1 X1^T and dP^T = Y2 X2^T on 16x16x32 MFMAs whose lanes hold
// one owned row and four streamed ones, which is the form the second products
// take P and dS in. P and dS are rounded to 16 bits there (the matrix cores' input
// type; with it gradients are 2.4e-3 off in bf16 where their own rounding leaves
// 1.7e-3), and so is out_rest, at most 2^-8 of the output; all sums are float32.
// Below 2^-14, a probability among 16,384 equal ones, fp16 has fewer bits: P is 2^10 P
// there until dV is stored. dS is as large as dO makes it and stays as it is.
// The first keys (sinks) are seen by every later query. Their tiles would run
// many times longer than the others, so their queries are split into parts whose
// float32 sums a third kernel adds up, always in the same order; so are all tiles of
// calls with too few of them to fill the chip.
// What bounds it: the matrix cores at the power limit and the LDS, whose operand
// reads (one 1 KiB fragment for two MFMAs) take as long as they do. 12 heads of
// 32,760 tokens, window of four frames of 1,560: keys 2,645 us (1,070 TFLOP/s over
// four products), queries 1,804 (1,180 over three), deltas 49, sinks 29. One
// kernel with the five products alone would have to add dQ up with atomics, in an
// order of its own each time.
#include <algorithm>
#include <initializer_list>

#include "window.hpp"

namespace ab {
namespace {

constexpr int kTileRows = kWindowKeys;  // streamed rows of a tile
constexpr int kStages = 4;              // of streamed tiles in LDS
constexpr int64_t kMostPartial = int64_t(1) << 28;  // floats
template <int D, bool kKeys>
constexpr int grad_lds() {
    return 2 * kStages * kTileRows * D * 2 + (kKeys ? kStages * 4 * 256 : 0);
}
static_assert(kTileRows == 32, "stat blocks are 32 queries");

template <class T>
constexpr float kLowered = 1.0f / (1 << T::kLift);

__device__ __forceinline__ int length_of(const WindowGradCall& c, int b) {
    return c.lengths ? min(max(c.lengths[b], 0), c.tokens) : c.tokens;
}

// stat of 32 queries of a head per workgroup: row r's normaliser (less kLift) and -delta, of the
// output before it was rounded (out + out_rest): with out alone dQ and dK of 4 x
// 4,099 tokens were 2.6e-3 off in bf16, 1.5 times the least that rounding them
// leaves (with logits of a deviation of 2, fp16: 3.12e-4 where rounding dS and dQ
// leaves 3.0e-4, and 3.08e-4 since out_rest makes up for the rounding of P's sum too).
// Rows past the batch item's length get zeros: nothing of theirs is read.
template <class T, int D>
__global__ __launch_bounds__(256) void window_delta_kernel(WindowGradCall c, int blocks) {
    constexpr int kLanes = D / 8, kRowsEach = 256 / kLanes;  // lanes of a row, rows at once
    const int bh = blockIdx.y + gridDim.y * blockIdx.z, b = bh / c.heads, h = bh - b * c.heads;
    if (b >= c.batch) return;
    const int length = length_of(c, b), lane = threadIdx.x % kLanes;
    float* stat = c.stat + (int64_t(bh) * blocks + blockIdx.x) * 64;
#pragma unroll
    for (int r = threadIdx.x / kLanes; r < 32; r += kRowsEach) {
        const int t = blockIdx.x * 32 + r;
        float sum = 0.f, lse = 0.f;
        if (t < length) {
            const uint16_t* o = static_cast<const uint16_t*>(c.out) + b * c.out_rows.batch + h * c.out_rows.head + t * c.out_rows.token;
            const uint16_t* d = static_cast<const uint16_t*>(c.dout) + b * c.dout_rows.batch + h * c.dout_rows.head + t * c.dout_rows.token;
            const u32x4 ow = *reinterpret_cast<const u32x4*>(o + 8 * lane), dw = *reinterpret_cast<const u32x4*>(d + 8 * lane);
            u32x4 rw = {0, 0, 0, 0};
            if (c.out_rest)
                rw = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(c.out_rest) + (o - static_cast<const uint16_t*>(c.out)) + 8 * lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum = __builtin_fmaf(T::lo(ow[i]) + T::lo(rw[i]), T::lo(dw[i]), sum);
                sum = __builtin_fmaf(T::hi(ow[i]) + T::hi(rw[i]), T::hi(dw[i]), sum);
            }
        }
#pragma unroll
        for (int s = 1; s < kLanes; s *= 2) sum += __shfl_xor(sum, s);
        if (t < length && lane == 0) {
            const int64_t at = int64_t(bh) * c.tokens + t;
            lse = c.lse[at] - T::kLift;
            if (c.dlse) sum -= c.dlse[at] * 1.4426950408889634f;
        }
        if (lane == 0) {
            stat[r] = lse;
            stat[32 + r] = -sum;
        }
    }
}

// 4 bytes per lane from the buffer straight into LDS: lane j writes [lds + 4j, + 4).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void buffer_to_lds4(u32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// A tensor's rows of one head, up to `rows` of them: reads past them give zeros.
template <int D>
__device__ __forceinline__ u32x4 head_buffer(const void* base, const Rows& r, int64_t b, int64_t h, int rows) {
    const char* at = static_cast<const char*>(base) + (b * r.batch + h * r.head) * 2;
    return buffer_of(at, rows > 0 ? static_cast<uint32_t>(rows - 1) * static_cast<uint32_t>(r.token * 2) + 2 * D : 0);
}

template <class T, int D, bool kKeys>
__global__ __launch_bounds__(kWindowThreads, 2) void window_grad_kernel(WindowGradCall c, WindowGrid places) {
    constexpr int kSteps = D / 32, kBlocks = D / 16, kQuad = 4 * D * 2, kBytes = kTileRows * D * 2, kOps = D / 64;
    constexpr int kOpRows = 1024 / (2 * D);
    // Four stages of Y1, four of Y2, and each wave's copy of the streamed rows' stat.
    constexpr int kY2 = kStages * kBytes, kStat = 2 * kStages * kBytes;
    extern __shared__ __align__(16) unsigned char smem[];
    touch(c.q, c.k_rows.batch, c.out_rows.batch, c.dq_rows.batch, c.lengths, c.partial);

    // Owned rows. Of keys, the sinks' tiles come first, part by part: `places` are
    // the tiles behind them. slot: the place of a part's sums.
    constexpr int kPartial = (kKeys ? 2 : 1) * kWindowRows * D;
    int head, tile, part = 0, parts = 1;
    uint32_t slot = blockIdx.x;
    if constexpr (kKeys) {
        const uint32_t split = c.batch * c.kv_heads * c.sink_tiles * c.sink_parts;
        if (blockIdx.x < split) {
            parts = c.sink_parts;
            tile = blockIdx.x / parts;
            part = blockIdx.x - tile * parts;
            head = tile / c.sink_tiles;
            tile -= head * c.sink_tiles;
        } else {
            const uint32_t id = (blockIdx.x - split) / c.key_parts;
            parts = c.key_parts;
            part = blockIdx.x - split - id * parts;
            places.place(id, head, tile);
            tile = places.tiles - 1 - tile;  // the first keys are seen most
            slot = split + (head * places.tiles + tile) * parts + part;
            tile += c.sink_tiles;
        }
    } else {
        const uint32_t id = blockIdx.x / c.query_parts;
        parts = c.query_parts;
        part = blockIdx.x - id * parts;
        places.place(id, head, tile);
        slot = (head * places.tiles + tile) * parts + part;
    }
    // Divisions leave them in vector registers.
    for (int* p : {&head, &tile, &part}) *p = __builtin_amdgcn_readfirstlane(*p);
    slot = __builtin_amdgcn_readfirstlane(slot);
    const int heads = kKeys ? c.kv_heads : c.heads;
    const int b = __builtin_amdgcn_readfirstlane(head / heads), h = head - b * heads;  // own head
    const int length = length_of(c, b);
    const WindowMask mask = c.mask;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    // The lane, for values made anew in each tile: D = 128 leaves the loop over
    // queries no register to keep them in (four spilled ones cost 10 %).
    auto lane_now = [&]() {
        int l = lane;
        asm volatile("" : "+v"(l));
        return l;
    };
    const int own0 = tile * kWindowRows, own_last = min(own0 + kWindowRows, length) - 1;

    // Queries that see a key at position p: start(p) .. until(p) - 1.
    auto until = [&](int p) {
        if (p < mask.sinks) return length;
        const uint32_t far = static_cast<uint32_t>(mask.start(p)) + mask.frame.d;
        return static_cast<int>(min(static_cast<uint32_t>(length), far + static_cast<uint32_t>(mask.back)));
    };

    // Streamed tiles: `rounds` heads times `tiles` tiles.
    TileRange range;
    int rounds = 1;
    if constexpr (kKeys) {
        range.sink_tiles = range.window = range.tiles = range.end = 0;
        if (own_last >= own0) {
            range.window = mask.start(own0) & ~(kTileRows - 1);
            range.end = own0 < mask.sinks ? length : until(own_last);
            range.tiles = (range.end - range.window + kTileRows - 1) / kTileRows;
        }
        rounds = c.group;
    } else {
        range.set(mask, own0, own_last, length);
    }
    const int64_t all = int64_t(rounds) * range.tiles;
    const int first = static_cast<int>(all * part / parts), last = static_cast<int>(all * (part + 1) / parts);

    // X as the B operand: owned row 16j + li of the wave's 32, dims 32s + 8lg .. + 7.
    u32x4 x1[2][kSteps], x2[2][kSteps];
    float lse[2] = {0.f, 0.f}, neg_delta[2] = {0.f, 0.f};
    const int stat_blocks = (c.tokens + 31) / 32;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int p = own0 + wave * 32 + 16 * j + li;
        const bool there = p < length;
        const int64_t at = min(p, c.tokens - 1);
        const Rows &r1 = kKeys ? c.k_rows : c.q_rows, &r2 = kKeys ? c.v_rows : c.dout_rows;
        const uint16_t* a = static_cast<const uint16_t*>(kKeys ? c.k : c.q) + b * r1.batch + h * r1.head + at * r1.token + 8 * lg;
        const uint16_t* d = static_cast<const uint16_t*>(kKeys ? c.v : c.dout) + b * r2.batch + h * r2.head + at * r2.token + 8 * lg;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            x1[j][s] = x2[j][s] = u32x4{0, 0, 0, 0};
            if (there) {
                x1[j][s] = *reinterpret_cast<const u32x4*>(a + 32 * s);
                x2[j][s] = *reinterpret_cast<const u32x4*>(d + 32 * s);
            }
        }
        if constexpr (!kKeys) {
            if (there) {
                const float* stat = c.stat + (int64_t(head) * stat_blocks + (p >> 5)) * 64 + (p & 31);
                lse[j] = stat[0] + T::kLift;
                neg_delta[j] = stat[32];
            }
        }
    }
    // Streamed rows that the owned row at p sees: from .. from + count - 1, and those
    // before sink.
    auto seen_rows = [&](int p, int& from, int& count, int& sink) {
        const bool there = p < length;
        if constexpr (kKeys) {
            from = mask.start(p);
            count = there ? until(p) - from : 0;
            sink = 0;
        } else {
            const int high = mask.high(p, length);
            from = mask.low(p);
            count = there ? high - from : 0;
            sink = there ? min(mask.sinks, high) : 0;
        }
    };
    // Tiles that all rows of this wave see whole need no mask.
    int full_from = 1, full_to = 0, full_sink = 0;
    const int w0 = own0 + wave * 32, w1 = min(w0 + 31, length - 1);
    const bool active = w1 >= w0;
    if (active) {
        if constexpr (kKeys) {
            full_from = mask.start(w1);
            full_to = w1 < mask.sinks ? length : until(max(w0, mask.sinks));
        } else {
            full_from = mask.low(w1);
            full_to = mask.high(w0, length);
            full_sink = min(mask.sinks, full_to);
        }
    }

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)smem));
    const Rows &y1_rows = kKeys ? c.q_rows : c.k_rows, &y2_rows = kKeys ? c.dout_rows : c.v_rows;
    const uint32_t y1_token = static_cast<uint32_t>(y1_rows.token * 2), y2_token = static_cast<uint32_t>(y2_rows.token * 2);
    // Transfers of this wave: rows 8w .. 8w + 7 of a tile. Every four rows lie as
    // blocks of 4 rows x 16 dims, block m at position m ^ (quad & 1): row reads and
    // transposing reads both spread over the banks.
    // With D = 128 a transfer is one quad, and the second one's blocks are swapped in
    // pairs: 32 bytes up or down.
    const int quad0 = D == 128 ? 0 : lane >> 5, block0 = (lane >> 3) % kBlocks;
    const uint32_t src_row = 8 * wave + 4 * quad0 + ((lane >> 1) & 3), src_at = (2 * (block0 ^ quad0) + (lane & 1)) * 16u;
    const uint32_t src1 = src_row * y1_token + src_at, src2 = src_row * y2_token + src_at;
    // The round and the tile of the next transfer.
    int next = first, next_round = range.tiles ? first / range.tiles : 0, next_tile = first - next_round * range.tiles;
    u32x4 y1_buf, y2_buf, stat_buf;
    auto enter_round = [&](int round) {
        const int hy = kKeys ? h * c.group + round : h / c.group;
        y1_buf = head_buffer<D>(kKeys ? c.q : c.k, y1_rows, b, hy, range.end);
        y2_buf = head_buffer<D>(kKeys ? c.dout : c.v, y2_rows, b, hy, range.end);
        if constexpr (kKeys)
            stat_buf = buffer_of(c.stat + (int64_t(b) * c.heads + hy) * stat_blocks * 64, stat_blocks * 256);
    };
    enter_round(next_round);
    auto transfer = [&]() {
        const uint32_t row = range.key(next_tile), place = next & (kStages - 1), stage = place * kBytes + wave * (8 * D * 2);
        // Past the last tile: nothing but the count.
        u32x4 y1 = y1_buf, y2 = y2_buf;
        if (next >= last) y1[2] = y2[2] = 0;
        if constexpr (kOps == 2) {
            const uint32_t swap = lane_now() & 8 ? -32 : 32;
            buffer_to_lds(y1, src1 + row * y1_token, src1 + swap + (row + kOpRows) * y1_token, lds0 + stage);
            buffer_to_lds(y2, src2 + row * y2_token, src2 + swap + (row + kOpRows) * y2_token, lds0 + kY2 + stage);
        } else {
            buffer_to_lds(y1, src1 + row * y1_token, lds0 + stage);
            buffer_to_lds(y2, src2 + row * y2_token, lds0 + kY2 + stage);
        }
        if constexpr (kKeys) {
            u32x4 stat = stat_buf;
            if (next >= last) stat[2] = 0;
            buffer_to_lds4(stat, row * 8 + 4 * lane_now(), lds0 + kStat + (place * 4 + wave) * 256);
        }
        ++next;
        if (++next_tile == range.tiles) {
            next_tile = 0;
            if (next < last) enter_round(++next_round);
        }
    };

    // Row reads (A of S and dP): row 16h + li, dims 32s + 8lg .. + 7: quad li / 4,
    // block 2s + lg / 2. Transposing reads as in the forward pass.
    uint32_t row_abs, tr_abs[2];
    {
        const int quad = li >> 2, par = quad & 1, base = quad * kQuad + (li & 3) * 32 + (lg & 1) * 16;
        // block m = 2s + lg / 2 at position m ^ par
        row_abs = lds0 + base + (((lg >> 1) ^ par)) * 128;
        const int tpar = lg & 1, tbase = lg * kQuad + 32 * (li >> 2) + 8 * (li & 3);
        tr_abs[0] = lds0 + tbase + tpar * 128;
        tr_abs[1] = lds0 + tbase - tpar * 128;
    }

    f32x4 acc1[kBlocks][2], acc2[kKeys ? kBlocks : 1][2];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            acc1[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (kKeys) acc2[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

    int tile_now = next_tile;
    if (first < last) {
        landed_and_barrier<0>();
        transfer();
        transfer();
        transfer();
    }
    // Stage t + 3 is that of t - 1, which every wave has left at the barrier.
    constexpr int kTileOps = 2 * kOps + (kKeys ? 1 : 0);
    for (int t = first; t < last; ++t) {
        landed_and_barrier<2 * kTileOps>();
        transfer();
        const int row0 = range.key(tile_now), place = t & (kStages - 1), stage = place * kBytes;
        if (++tile_now == range.tiles) tile_now = 0;
        if (!active) continue;
        const bool masked = !((row0 >= full_from && row0 + kTileRows <= full_to) || row0 + kTileRows <= full_sink);

        // In halves of 16 streamed rows: S and dP of row 16 half + 4lg + r and owned
        // row 16j + li, then P and dS as the second products take them.
        u32x4 pw[2], dw[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 sc[2], dp[2], row_lse;
            if constexpr (kKeys) {
                const uint32_t at = lds0 + kStat + (place * 4 + wave) * 256 + 64 * half + 16 * (lane_now() >> 4);
                row_lse = __builtin_bit_cast(f32x4, lds_read16(at));
                dp[0] = dp[1] = __builtin_bit_cast(f32x4, lds_read16(at + 128));
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (!kKeys) dp[j] = f32x4{neg_delta[j], neg_delta[j], neg_delta[j], neg_delta[j]};
            }
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const u32x4 a1 = lds_read16(row_abs + stage + half * 4 * kQuad + s * 256);
                const u32x4 a2 = lds_read16(row_abs + stage + kY2 + half * 4 * kQuad + s * 256);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    sc[j] = T::mfma16(a1, x1[j][s], sc[j]);
                    dp[j] = T::mfma16(a2, x2[j][s], dp[j]);
                }
            }
            // sc becomes P, dp dS.
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    sc[j][r] = fast_exp2(__builtin_fmaf(sc[j][r], c.scale_log2, kKeys ? -row_lse[r] : -lse[j]));
                    if constexpr (kKeys && T::kLift > 0) dp[j][r] *= kLowered<T>;
                    dp[j][r] *= sc[j][r];
                }
            if (masked) {
                const int l = lane_now(), row = row0 + 16 * half + 4 * (l >> 4);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    int from, count, sink;
                    seen_rows(own0 + wave * 32 + 16 * j + (l & 15), from, count, sink);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        bool sees = static_cast<uint32_t>(row + r - from) < static_cast<uint32_t>(count);
                        if constexpr (!kKeys) sees |= row + r < sink;
                        sc[j][r] = sees ? sc[j][r] : 0.f;
                        dp[j][r] = sees ? dp[j][r] : 0.f;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    pw[j][2 * half + r / 2] = T::pack(sc[j][r], sc[j][r + 1]);
                    dw[j][2 * half + r / 2] = T::pack(dp[j][r], dp[j][r + 1]);
                }
            // Reads of the next half not before: with them D = 128 spills.
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
            const uint32_t at = tr_abs[m & 1] + stage + m * 128;
            const u32x4 a1 = __builtin_bit_cast(u32x4, __builtin_shufflevector(lds_read_transposed(at), lds_read_transposed(at + 4 * kQuad), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int j = 0; j < 2; ++j) acc1[m][j] = T::mfma16(a1, dw[j], acc1[m][j]);
            if constexpr (kKeys) {
                const u32x4 a2 = __builtin_bit_cast(u32x4, __builtin_shufflevector(lds_read_transposed(at + kY2), lds_read_transposed(at + kY2 + 4 * kQuad), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int j = 0; j < 2; ++j) acc2[m][j] = T::mfma16(a2, pw[j], acc2[m][j]);
            }
        }
    }

    // No transfer may still be landing when the LDS is released.
    landed_and_barrier<0>();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int p = own0 + wave * 32 + 16 * j + li;
        if (parts > 1) {
            float* dst = c.partial + int64_t(slot) * kPartial + (p - own0) * D + 4 * lg;
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                *reinterpret_cast<f32x4*>(dst + 16 * m) = acc1[m][j];
                if constexpr (kKeys) *reinterpret_cast<f32x4*>(dst + kWindowRows * D + 16 * m) = acc2[m][j];
            }
            continue;
        }
        if (p >= c.tokens) continue;
        const float live = p < length ? 1.f : 0.f;
        const Rows& r1 = kKeys ? c.dk_rows : c.dq_rows;
        uint16_t* d1 = static_cast<uint16_t*>(kKeys ? c.dk : c.dq) + b * r1.batch + h * r1.head + p * r1.token + 4 * lg;
        const float scale = c.scale;
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
            f32x4 g = acc1[m][j] * scale;
            if (live == 0.f) g = f32x4{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<u32x2*>(d1 + 16 * m) = u32x2{T::pack(g[0], g[1]), T::pack(g[2], g[3])};
        }
        if constexpr (kKeys) {
            uint16_t* d2 = static_cast<uint16_t*>(c.dv) + b * c.dv_rows.batch + h * c.dv_rows.head + p * c.dv_rows.token + 4 * lg;
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                f32x4 g = acc2[m][j] * kLowered<T>;
                if (live == 0.f) g = f32x4{0.f, 0.f, 0.f, 0.f};
                *reinterpret_cast<u32x2*>(d2 + 16 * m) = u32x2{T::pack(g[0], g[1]), T::pack(g[2], g[3])};
            }
        }
    }
}

// The parts of split tiles added up, in order: eight values of a row per thread.
// Tiles first .. first + count - 1 of every head; outputs dK and dV, or dQ alone.
struct Sums {
    const float* partial;
    int first, count, parts, heads, outputs;
    void* out[2];
    Rows rows[2];
    float scale[2];
};
template <class T, int D>
__global__ __launch_bounds__(256) void window_sums_kernel(WindowGradCall c, Sums s) {
    constexpr int kLanes = D / 8, kTileValues = kWindowRows * D;
    const int at = blockIdx.x * 256 + threadIdx.x;  // of a tile's rows times lanes, of the first output, then of the second
    const int which = at / (kWindowRows * kLanes), row = at / kLanes % kWindowRows, lane = at % kLanes;
    const int head = blockIdx.z, b = head / s.heads, h = head - b * s.heads;
    const int p = (s.first + static_cast<int>(blockIdx.y)) * kWindowRows + row;
    if (which >= s.outputs || p >= c.tokens) return;
    float sum[8] = {};
    if (p < length_of(c, b)) {
        const int64_t each = int64_t(s.outputs) * kTileValues;
        const float* src = s.partial + (int64_t(head) * s.count + blockIdx.y) * s.parts * each + which * kTileValues + row * D + lane * 8;
        for (int i = 0; i < s.parts; ++i, src += each) {
            const f32x4 x = reinterpret_cast<const f32x4*>(src)[0], y = reinterpret_cast<const f32x4*>(src)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[e] += x[e];
                sum[4 + e] += y[e];
            }
        }
    }
    const float scale = which ? s.scale[1] : s.scale[0];
    const Rows r = which ? s.rows[1] : s.rows[0];
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = T::pack(sum[2 * i] * scale, sum[2 * i + 1] * scale);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(which ? s.out[1] : s.out[0]) + b * r.batch + h * r.head + p * r.token + lane * 8) = w;
}

template <class T, int D>
int launch_as(const WindowGradCall& c, hipStream_t stream) {
    const int blocks = (c.tokens + 31) / 32, tiles = (c.tokens + kWindowRows - 1) / kWindowRows;
    const unsigned bh = static_cast<unsigned>(c.batch * c.heads), kv = static_cast<unsigned>(c.batch * c.kv_heads);
    const unsigned y = std::min(bh, 32768u);
    hipLaunchKernelGGL((window_delta_kernel<T, D>), dim3(blocks, y, (bh + y - 1) / y), dim3(256), 0, stream, c, blocks);
    if (int rc = check_launch("window_delta_kernel")) return rc;
    auto sums = [&](const Sums& s, unsigned all_heads) {
        hipLaunchKernelGGL((window_sums_kernel<T, D>), dim3(s.outputs * kWindowRows * (D / 8) / 256, s.count, all_heads), dim3(256), 0,
                           stream, c, s);
        return check_launch("window_sums_kernel");
    };
    const unsigned split = kv * c.sink_tiles * c.sink_parts;
    const WindowGrid keys = window_grid(kv, tiles - c.sink_tiles), queries = window_grid(bh, tiles);
    const auto by_keys = window_grad_kernel<T, D, true>, by_queries = window_grad_kernel<T, D, false>;
    if (int rc = ensure_lds_limit(reinterpret_cast<const void*>(by_keys), grad_lds<D, true>())) return rc;
    if (int rc = ensure_lds_limit(reinterpret_cast<const void*>(by_queries), grad_lds<D, false>())) return rc;
    hipLaunchKernelGGL(by_keys, dim3(split + keys.size() * c.key_parts), dim3(kWindowThreads), (grad_lds<D, true>()), stream, c, keys);
    if (int rc = check_launch("window_grad_kernel")) return rc;
    Sums s{c.partial, 0, c.sink_tiles, c.sink_parts, c.kv_heads, 2, {c.dk, c.dv}, {c.dk_rows, c.dv_rows}, {c.scale, kLowered<T>}};
    if (c.sink_tiles)
        if (int rc = sums(s, kv)) return rc;
    const int64_t each = int64_t(kWindowRows) * D;
    s.partial += int64_t(split) * 2 * each;
    s.first = c.sink_tiles;
    s.count = static_cast<int>(keys.tiles);
    s.parts = c.key_parts;
    if (c.key_parts > 1)
        if (int rc = sums(s, kv)) return rc;
    WindowGradCall q = c;
    if (c.key_parts > 1) s.partial += int64_t(keys.size()) * c.key_parts * 2 * each;
    q.partial = const_cast<float*>(s.partial);
    hipLaunchKernelGGL(by_queries, dim3(queries.size() * c.query_parts), dim3(kWindowThreads), (grad_lds<D, false>()), stream, q, queries);
    if (int rc = check_launch("window_grad_kernel")) return rc;
    if (c.query_parts == 1) return 0;
    return sums({q.partial, 0, tiles, c.query_parts, c.heads, 1, {c.dq, c.dq}, {c.dq_rows, c.dq_rows}, {c.scale, c.scale}}, bh);
}
}  // namespace

// Tiles with sinks are split into parts of about as many queries as a tile
// behind them has (its window), at most 64 of them and 1 GiB of partial sums. All
// tiles are split where that gives each CU at most two workgroups, of eight steps at
// least: 1,560 tokens of 4 heads over 2, 4 frames of 390: 224 us forward and backward
// with whole tiles, 95 with split ones.
void plan_window_grad(WindowGradCall& c, int64_t& stat, int64_t& partial) {
    const int64_t blocks = (int64_t(c.tokens) + 31) / 32, tiles = (int64_t(c.tokens) + kWindowRows - 1) / kWindowRows;
    stat = int64_t(c.batch) * c.heads * blocks * 64;
    partial = 0;
    c.sink_tiles = c.sink_parts = 0;
    c.key_parts = c.query_parts = 1;
    const int64_t window = int64_t(c.mask.back) + c.mask.frame.d + kWindowRows;
    const int64_t kv = int64_t(c.batch) * c.kv_heads, bh = int64_t(c.batch) * c.heads;
    const int64_t each = kWindowRows * int64_t(c.dim);  // floats of a part
    if (tiles > 65535 || bh > 65535) return;
    const int64_t sinks = std::min<int64_t>((int64_t(c.mask.sinks) + kWindowRows - 1) / kWindowRows, tiles);
    if (sinks > 0) {
        const int64_t parts = std::min<int64_t>({(c.tokens + window - 1) / window, 64, kMostPartial / (kv * sinks * 2 * each)});
        if (parts > 1) {
            c.sink_tiles = static_cast<int32_t>(sinks);
            c.sink_parts = static_cast<int32_t>(parts);
            partial = kv * sinks * parts * 2 * each;
        }
    }
    auto split = [&](int64_t units, int64_t steps) {
        // No units: the sinks' tiles are all there are.
        return units == 0 ? 1 : static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({512 / units, steps / 8, 16})));
    };
    const int64_t seen = std::min<int64_t>(window, c.tokens);  // queries of a key tile, about
    const int64_t key_units = kv * (tiles - c.sink_tiles), query_units = bh * tiles;
    c.key_parts = split(key_units, c.group * (seen / kTileRows));
    c.query_parts = split(query_units, std::min<int64_t>(seen + c.mask.sinks, c.tokens) / kTileRows);
    if (c.key_parts > 1) partial += key_units * c.key_parts * 2 * each;
    if (c.query_parts > 1) partial += query_units * c.query_parts * each;
}

int launch_window_grad(const WindowGradCall& c, hipStream_t stream) {
    if (c.dim == 128) return c.half ? launch_as<F16, 128>(c, stream) : launch_as<Bf16, 128>(c, stream);
    return c.half ? launch_as<F16, 64>(c, stream) : launch_as<Bf16, 64>(c, stream);
}

}  // namespace ab
