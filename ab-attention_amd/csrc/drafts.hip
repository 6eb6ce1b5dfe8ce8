// Drafted tokens: the lines of their tree, and which of them stay.
#include <initializer_list>

#include "drafts.hpp"

namespace ab {
namespace {

constexpr int kWave = 64;

// ---- the tree -----------------------------------------------------------------
//
// Token i of a sequence's n new ones is at position length - n + depth(i), where depth
// counts the drafts above it. Its line (the tokens above it, and itself) is kept in
// words of 64 places: the word of its own 64 and the last place before them, whose word
// goes on. A walk up a line takes a step for every 64 places, and every layer's
// attention reads 16 bytes a token.
//
// One workgroup per sequence, 256 tokens at a time, a lane each: every wave follows the lines
// inside its 64 by six rounds of pointer doubling (word, steps and end of a line twice as
// long each time) by lane exchanges; then the waves take the positions above theirs one after
// the other. Bound by launch and latency: in calls in a row 26 drafts 2.1 us, 4 x 701 4.2 (one
// wave for all of a sequence 7.6).
constexpr int kTreeWaves = 4;
__global__ __launch_bounds__(kWave * kTreeWaves) void tree_kernel(TreeCall c) {
    constexpr int kTokens = kWave * kTreeWaves;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int off = min(max(c.offsets[b], 0), c.tokens), n = min(max(c.offsets[b + 1], 0), c.tokens) - off;
    const int first = c.lengths[b] - n;
    // Rows of no sequence.
    auto clear = [&](int from, int to) {
        for (int i = from + static_cast<int>(threadIdx.x); i < to; i += kTokens) {
            c.positions[i] = 0;
            c.near[i] = 0;
            c.above[i] = -1;
        }
    };
    if (b == 0) clear(0, off);
    if (b == c.batch - 1) clear(off + max(n, 0), c.tokens);
    // Positions of earlier tokens; of those past what fits, what was written.
    constexpr int kNear = 4096;
    __shared__ int positions[kNear];
    for (int block0 = 0; block0 < n; block0 += kTokens) {
        const int block = block0 + wave * kWave, i = block + lane;
        int parent = i < n ? c.parents[off + i] : -1;
        if (parent >= i) parent = -1;
        const bool inside = parent >= block;
        uint64_t word = uint64_t(1) << lane;
        int end = inside ? parent - block : lane, steps = inside ? 1 : 0;
#pragma unroll
        for (int s = 0; s < 6; ++s) {
            const uint64_t its_word = __shfl(static_cast<unsigned long long>(word), end);
            const int its_steps = __shfl(steps, end), its_end = __shfl(end, end);
            word |= its_word;
            steps += its_steps;
            end = its_end;
        }
        const int above = max(__shfl(parent, end), -1);
        if (i < n) {
            c.near[off + i] = word;
            c.above[off + i] = above;
        }
        for (int w = 0; w < kTreeWaves && block0 + w * kWave < n; ++w) {
            if (wave == w && i < n) {
                int position = first + steps;
                if (above >= kNear) position = c.positions[off + above] + 1 + steps;
                else if (above >= 0) position = positions[above] + 1 + steps;
                if (i < kNear) positions[i] = position;
                c.positions[off + i] = position;
            }
            __threadfence_block();
            __syncthreads();
        }
    }
}

// ---- verification -------------------------------------------------------------
//
// The first new token of a sequence is kept. From the last kept token on its children j
// (tokens x_j) are looked at in the order of their places, with w what is left of the
// target's probabilities p behind it and S the sum that w counts by (w = p, S = 1 at
// first): j is kept, and becomes the last one, where
//   u_j q(x_j) S < w(x_j)        (q: the draft's probabilities; chosen drafts: q = 1)
// and else
//   drawn drafts:   w <- max(w - S q, 0), S <- sum of w (nothing changes where that is 0)
//   chosen drafts:  S <- S - w(x_j), w(x_j) <- 0.
// Where no child is left the next token is the first with w > 0 whose running sum of w
// passes u_0 times the whole sum. As q is not negative, w = max(p - c q, 0) with c the sum
// of the S so far: two numbers say what several turned down drafts have left. Sums and
// products are in 64 bits: a running sum over 100,000 tokens of nearly equal weights passes a
// border within its own float32 error in a hundredth of all calls. Values that are not
// positive and finite count as 0.
//
// Two kernels. verify_kernel: every workgroup walks down its sequence's tree as far as
// that needs no sum over the vocabulary (chosen drafts: to the end; drawn ones: to the
// first that is turned down), 64 drafts at a time in the lanes of a wave, whose p and q
// are fetched together before the first is looked at; then each of its waves adds up a
// part of what is left. sample_kernel, one workgroup per sequence, goes on from there:
// where more drawn drafts are turned down it adds up the whole vocabulary by itself.
//
// A chain of 7 drafts over 32,000 tokens takes 4.6 + 4.8 us, 48 chosen trees over 128,000
// 10.4 + 5.2, bound by latency: the walk, a reading, the choice among a few values. What
// one CU adds up by itself takes 2.3 us over 1,000 tokens, 4.1 over 32,000 and 8.9 over
// 100,000, as much 64-bit arithmetic as loading (16 drawn trees with four drafts behind a
// token, four or five such sums after one another: 5 + 40 us). A kernel for every further
// sum would spread them over the chip, and cost those that have none 2 us and a launch each.

// The value of an element, and its weight: of what is negative, infinite or no number 0.
// As unsigned numbers the bits of positive finite ones are those up to the largest one's.
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ float value_of(_Float16 x) { return static_cast<float>(x); }
constexpr uint32_t kLargest = 0x7f7fffffu;
template <class E>
__device__ __forceinline__ float weight_of(E x) {
    const float w = value_of(x);
    return __float_as_uint(w) <= kLargest ? w : 0.f;
}

__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ double from_halves(uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo); }
__device__ __forceinline__ uint32_t low_half(double x) { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, x)); }
__device__ __forceinline__ uint32_t high_half(double x) { return static_cast<uint32_t>(__builtin_bit_cast(uint64_t, x) >> 32); }
__device__ __forceinline__ double lane_value(double x, int lane) {
    return from_halves(__builtin_amdgcn_readlane(low_half(x), lane), __builtin_amdgcn_readlane(high_half(x), lane));
}
// x of the lane that a DPP control names, 0 where there is none.
template <int kControl>
__device__ __forceinline__ double moved(double x) {
    return from_halves(__builtin_amdgcn_update_dpp(0, low_half(x), kControl, 15, 15, true),
                       __builtin_amdgcn_update_dpp(0, high_half(x), kControl, 15, 15, true));
}
// The sum over the lanes, in all of them (a tenth of the time of exchanges through LDS).
__device__ __forceinline__ double lanes_sum(double x) {
    x += moved<0xb1>(x);   // quad_perm 1 0 3 2
    x += moved<0x4e>(x);   // quad_perm 2 3 0 1
    x += moved<0x141>(x);  // row_half_mirror
    x += moved<0x140>(x);  // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(low_half(x), low_half(x), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(high_half(x), high_half(x), false, false);
    x = from_halves(a[0], b[0]) + from_halves(a[1], b[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(low_half(x), low_half(x), false, false);
    const auto d = __builtin_amdgcn_permlane32_swap(high_half(x), high_half(x), false, false);
    return from_halves(c[0], d[0]) + from_halves(c[1], d[1]);
}
// x and those of the lanes before.
__device__ __forceinline__ double running_sum(double x, int lane) {
    x += moved<0x111>(x);  // row_shr 1, 2, 4, 8
    x += moved<0x112>(x);
    x += moved<0x114>(x);
    x += moved<0x118>(x);
    const double one = lane_value(x, 15), two = one + lane_value(x, 31), three = two + lane_value(x, 47);
    return x + (lane < 16 ? 0.0 : lane < 32 ? one : lane < 48 ? two : three);
}

constexpr int kEach = 8;  // neighbouring tokens of the vocabulary that a lane takes at a time
constexpr int kTimes = kVerifyStep / (kWave * kEach);

// A step of a row: x[i] are the tokens from at + i kWave kEach on, 0 behind the last one.
template <class E>
struct Step {
    E x[kTimes][kEach];
    __device__ __forceinline__ void read(const E* row, int step, int lane, int vocab) {
        const int at = step * kVerifyStep + lane * kEach;
        if ((step + 1) * kVerifyStep <= vocab) {  // the same in all lanes
#pragma unroll
            for (int i = 0; i < kTimes; ++i) __builtin_memcpy(x[i], row + at + i * kWave * kEach, sizeof(x[i]));
        } else {
            int from = at;
            asm volatile("" : "+v"(from));  // addresses are made here, not kept in registers for all steps
#pragma unroll
            for (int i = 0; i < kTimes; ++i)
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int token = from + i * kWave * kEach + e;
                    const E value = row[min(token, vocab - 1)];
                    x[i][e] = token < vocab ? value : E(0);
                }
        }
    }
    __device__ __forceinline__ void weights(float (&w)[kTimes][kEach]) const {
#pragma unroll
        for (int i = 0; i < kTimes; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) w[i][e] = weight_of(x[i][e]);
    }
    // The same where all are weights already; the largest of the values' bits with `top`.
    __device__ __forceinline__ uint32_t values(float (&w)[kTimes][kEach], uint32_t top) const {
#pragma unroll
        for (int i = 0; i < kTimes; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                w[i][e] = value_of(x[i][e]);
                top = max(top, __float_as_uint(w[i][e]));
            }
        return top;
    }
};

template <class E>
struct Verifier {
    const VerifyCall& c;
    int off, n, lane;
    // The 64 new tokens of a window, one to a lane: whom they follow, their token, p and
    // q u of it behind that one.
    int window = -1, parent, token;
    double p, uq, q;

    __device__ Verifier(const VerifyCall& call, int b) : c(call), lane(threadIdx.x & 63) {
        off = min(max(c.offsets[b], 0), c.rows);
        n = min(max(c.offsets[b + 1], 0), c.rows) - off;
    }
    __device__ __forceinline__ const E* target(int place) const {
        return static_cast<const E*>(c.target) + int64_t(off + place) * c.target_row;
    }
    __device__ __forceinline__ const E* draft(int place) const {
        return static_cast<const E*>(c.draft) + int64_t(off + place) * c.draft_row;
    }
    // -1 for none of the vocabulary.
    __device__ __forceinline__ int token_at(int place) const {
        const int64_t x = c.wide ? static_cast<const int64_t*>(c.tokens)[off + place] : static_cast<const int32_t*>(c.tokens)[off + place];
        return x >= 0 && x < c.vocab ? static_cast<int>(x) : -1;
    }

    __device__ __forceinline__ void look_at(int from) {
        if (from == window) return;
        window = from;
        const int place = from + lane;
        parent = token = -1;
        uq = 0.0;
        if (place < n) {
            parent = c.parents[off + place];
            token = token_at(place);
            uq = static_cast<double>(c.uniforms[off + place]);
        }
        if (parent >= place) parent = -1;
        const bool there = parent >= 0 && token >= 0;
        p = there ? static_cast<double>(weight_of(target(parent)[token])) : 0.0;
        q = 1.0;
        if (c.draft) {
            q = there ? static_cast<double>(weight_of(draft(parent)[token])) : 0.0;
            uq *= q;
        }
    }

    // Walks on from s, S = sum, until no child is left (true) or, among drawn drafts, one
    // has been turned down (false; not counted into s.less yet). All 64 lanes alike.
    __device__ bool walk(VerifyState& s, double& sum, bool writes) {
        for (int from = s.next & ~(kWave - 1); from < n; from += kWave) {
            look_at(from);
            for (;;) {
                const uint64_t left = __ballot(parent >= 0 && parent == s.last && from + lane >= s.next);
                if (left == 0) break;
                const int at = __builtin_ctzll(left);
                double size = lane_value(p, at);
                const double bar = lane_value(uq, at);
                if (c.draft) {
                    if (s.gone > 0) size = fmax(__builtin_fma(-s.less, lane_value(q, at), size), 0.0);
                } else if (s.gone > 0) {
                    // Chosen before: nothing is left of it.
                    const int its = lane_value(token, at);
                    bool again = __ballot(parent == s.last && token == its && lane < at) != 0;
                    for (int before = s.last + 1; before < from && !again; before += kWave) {
                        const int i = before + lane;
                        again = __ballot(i < from && c.parents[off + i] == s.last && token_at(i) == its) != 0;
                    }
                    if (again) size = 0.0;
                }
                s.next = from + at + 1;
                if (__builtin_amdgcn_readfirstlane(bar * sum < size)) {
                    s.last = from + at;
                    if (writes && lane == 0) c.path[off + s.counts] = s.last;
                    ++s.counts;
                    s.gone = 0;
                    s.less = 0.0;
                    sum = 1.0;
                } else {
                    if (c.draft) return false;
                    ++s.gone;
                    sum -= size;
                }
            }
        }
        return true;
    }

    // Chosen drafts behind the last kept token: nothing is left of them. w are the weights of
    // the tokens from `at` on.
    __device__ __forceinline__ void take_chosen(const VerifyState& s, int at, float (&w)[kTimes][kEach]) const {
        for (int from = (s.last + 1) & ~(kWave - 1); from < n; from += kWave) {
            const int place = from + lane;
            const int x = place < n && place > s.last && c.parents[off + place] == s.last ? token_at(place) : -1;
            for (uint64_t gone = __ballot(x >= 0); gone; gone &= gone - 1) {
                const int its = lane_value(x, __builtin_ctzll(gone));
#pragma unroll
                for (int i = 0; i < kTimes; ++i)
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        if (its == at + i * kWave * kEach + e) w[i][e] = 0.f;
            }
        }
    }

    // What is left of a step's tokens.
    __device__ __forceinline__ void left_of(const VerifyState& s, int step, double (&left)[kTimes][kEach]) const {
        Step<E> ps, qs;
        float w[kTimes][kEach];
        ps.read(target(s.last), step, lane, c.vocab);
        ps.weights(w);
        if (!c.draft && s.gone > 0) take_chosen(s, step * kVerifyStep + lane * kEach, w);
#pragma unroll
        for (int i = 0; i < kTimes; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) left[i][e] = static_cast<double>(w[i][e]);
        if (!c.draft || s.gone == 0) return;
        qs.read(draft(s.last), step, lane, c.vocab);
        qs.weights(w);
#pragma unroll
        for (int i = 0; i < kTimes; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) left[i][e] = fmax(__builtin_fma(-s.less, static_cast<double>(w[i][e]), left[i][e]), 0.0);
    }

    // The sums of the parts first, first + stride, ..: one to a wave, written by its lane 0.
    // kDrawn: drawn drafts have been turned down. A step costs a lane five operations in 64
    // bits and one and a half others for each token; values that are no weights, which are found
    // by the largest of the bits, cost two more.
    template <bool kDrawn>
    __device__ __forceinline__ void add_up_as(const VerifyState& s, int first, int stride, double* sums) const {
        const E *row = target(s.last), *less_row = kDrawn ? draft(s.last) : nullptr;
        const double less = s.less;
        const bool chosen = !c.draft && s.gone > 0;
        Step<E> ps, qs;
        auto read = [&](int step) {
            ps.read(row, step, lane, c.vocab);
            if (kDrawn) qs.read(less_row, step, lane, c.vocab);
        };
        if (first < c.parts) read(first * c.times);
        for (int part = first; part < c.parts; part += stride) {
            double sum = 0.0, odd = 0.0;
            const int end = min((part + 1) * c.times, (c.vocab + kVerifyStep - 1) / kVerifyStep);
            for (int step = part * c.times; step < end; ++step) {
                float p[kTimes][kEach], q[kTimes][kEach];
                uint32_t top = ps.values(p, 0);
                if (kDrawn) top = qs.values(q, top);
                if (__ballot(top > kLargest)) {
                    ps.weights(p);
                    if (kDrawn) qs.weights(q);
                }
                // The next step is on its way while this one is added up.
                if (step + 1 < end) read(step + 1);
                else if (part + stride < c.parts) read((part + stride) * c.times);
                if (!kDrawn && chosen) take_chosen(s, step * kVerifyStep + lane * kEach, p);
#pragma unroll
                for (int i = 0; i < kTimes; ++i)
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        const double w = static_cast<double>(p[i][e]);
                        (e & 1 ? odd : sum) += kDrawn ? fmax(__builtin_fma(-less, static_cast<double>(q[i][e]), w), 0.0) : w;
                    }
            }
            sum = lanes_sum(sum + odd);
            if (lane == 0) sums[part] = sum;
        }
    }
    __device__ __forceinline__ void add_up(const VerifyState& s, int first, int stride, double* sums) const {
        if (c.draft && s.gone > 0) add_up_as<true>(s, first, stride, sums);
        else add_up_as<false>(s, first, stride, sums);
    }
};

template <class E>
__global__ __launch_bounds__(256) void verify_kernel(VerifyCall c) {
    const int b = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Verifier<E> v(c, b);
    if (v.n <= 0) return;
    const bool writes = blockIdx.x == 0 && wave == 0;
    VerifyState s{0.0, 0, 1, 1, 0};
    double sum = 1.0;
    if (!v.walk(s, sum, writes)) {
        s.less = 1.0;
        s.gone = 1;
    }
    if (writes && v.lane == 0) c.state[b] = s;
    v.add_up(s, blockIdx.x * 4 + wave, c.parts, c.sums + int64_t(b) * c.parts);
}

constexpr int kSampleWaves = 16;

template <class E>
__global__ __launch_bounds__(kSampleWaves * kWave) void sample_kernel(VerifyCall c) {
    __shared__ double sums[kVerifyParts];
    __shared__ VerifyState known;
    __shared__ int go_on;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Verifier<E> v(c, b);
    // Rows of no sequence have no path.
    if (b == 0)
        for (int i = threadIdx.x; i < v.off; i += blockDim.x) c.path[i] = -1;
    if (b == c.batch - 1)
        for (int i = v.off + max(v.n, 0) + threadIdx.x; i < c.rows; i += blockDim.x) c.path[i] = -1;
    auto finish = [&](int counts, int next) {
        c.counts[b] = counts;
        if (c.wide) static_cast<int64_t*>(c.next)[b] = next;
        else static_cast<int32_t*>(c.next)[b] = next;
    };
    if (v.n <= 0) {
        if (threadIdx.x == 0) finish(0, -1);
        return;
    }
    VerifyState s = c.state[b];
    for (int32_t* x : {&s.last, &s.next, &s.counts, &s.gone}) *x = __builtin_amdgcn_readfirstlane(*x);
    if (threadIdx.x < c.parts) sums[threadIdx.x] = c.sums[int64_t(b) * c.parts + threadIdx.x];
    __syncthreads();
    // The first wave decides, all of them add up.
    double total = 0.0, sum = 1.0, less = 0.0;  // S and c before the draft that was turned down last
    bool walked = !c.draft || s.gone == 0;
    for (;;) {
        if (wave == 0) {
            total = 0.0;
            for (int p = lane; p < c.parts; p += kWave) total += sums[p];
            total = lanes_sum(total);
            bool more = false;
            if (!walked) {
                // total is the sum of what the draft that was turned down last has left.
                const bool some = __builtin_amdgcn_readfirstlane(total > 0.0) != 0;
                if (some) {
                    sum = total;
                } else {  // nothing: it changes nothing
                    s.less = less;
                    --s.gone;
                }
                const int counts = s.counts;
                walked = v.walk(s, sum, true);
                less = s.less;
                if (!walked) {
                    s.less += sum;
                    ++s.gone;
                }
                more = !walked || !some || s.counts != counts;
            }
            if (lane == 0) {
                known = s;
                go_on = more;
            }
        }
        __syncthreads();
        if (wave > 0) s = known;
        if (!go_on) break;
        for (int32_t* x : {&s.last, &s.gone}) *x = __builtin_amdgcn_readfirstlane(*x);
        v.add_up(s, wave, kSampleWaves, sums);
        __syncthreads();
    }
    // The next token.
    for (int i = s.counts + threadIdx.x; i < v.n; i += blockDim.x) c.path[v.off + i] = -1;
    if (wave != 0) return;
    if (lane == 0) c.path[v.off] = 0;
    const double border = static_cast<double>(c.uniforms[v.off]) * total;
    // The part where the running sum passes the border, or the last one with a weight.
    double before = 0.0, base = 0.0;
    int part = -1;
    bool past = false;
    for (int p = 0; p < c.parts && !past; p += kWave) {
        const double own = p + lane < c.parts ? sums[p + lane] : 0.0, run = running_sum(own, lane);
        const uint64_t passes = __ballot(own > 0.0 && before + run > border), has = __ballot(own > 0.0);
        past = passes != 0;
        if (has) {
            const int at = past ? __builtin_ctzll(passes) : 63 - __builtin_clzll(has);
            part = p + at;
            base = before + (at > 0 ? lane_value(run, at - 1) : 0.0);
        }
        before += lane_value(run, kWave - 1);
    }
    int found = -1;  // the token in it, likewise
    past = false;
    for (int t = 0; part >= 0 && t < c.times && !past; ++t) {
        const int step = part * c.times + t;
        double w[kTimes][kEach];
        v.left_of(s, step, w);
#pragma unroll
        for (int i = 0; i < kTimes; ++i) {
            double own = 0.0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) own += w[i][e];
            const double run = running_sum(own, lane), until = __shfl_up(run, 1);
            double at = base + (lane == 0 ? 0.0 : until);
            int first = -1, any = -1;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                at += w[i][e];
                if (w[i][e] > 0.0) {
                    any = e;
                    if (first < 0 && at > border) first = e;
                }
            }
            const uint64_t passes = __ballot(first >= 0), has = __ballot(any >= 0);
            if (has && !past) {
                past = passes != 0;
                found = lane_value(step * kVerifyStep + (i * kWave + lane) * kEach + (past ? first : any),
                                   past ? __builtin_ctzll(passes) : 63 - __builtin_clzll(has));
            }
            base += lane_value(run, kWave - 1);
        }
    }
    if (lane == 0) finish(s.counts, found);
}

template <class E>
int launch_verify_as(const VerifyCall& c, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((c.parts + 3) / 4), static_cast<unsigned>(c.batch));
    hipLaunchKernelGGL(verify_kernel<E>, grid, dim3(256), 0, stream, c);
    if (int rc = check_launch("verify_kernel")) return rc;
    hipLaunchKernelGGL(sample_kernel<E>, dim3(static_cast<unsigned>(c.batch)), dim3(kSampleWaves * kWave), 0, stream, c);
    return check_launch("sample_kernel");
}
}  // namespace

int launch_tree(const TreeCall& c, hipStream_t stream) {
    hipLaunchKernelGGL(tree_kernel, dim3(static_cast<unsigned>(c.batch)), dim3(kWave * kTreeWaves), 0, stream, c);
    return check_launch("tree_kernel");
}

int launch_verify(const VerifyCall& c, hipStream_t stream) {
    return c.type == 0 ? launch_verify_as<uint16_t>(c, stream)
         : c.type == 1 ? launch_verify_as<_Float16>(c, stream) : launch_verify_as<float>(c, stream);
}

}  // namespace ab
