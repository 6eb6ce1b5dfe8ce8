// Drafted tokens: the lines of their tree, and which of them stay.
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
// One wave per sequence, 64 tokens at a time, a lane each: six rounds of pointer
// doubling (word, steps and end of a line twice as long each time) by lane exchanges. Bound by
// launch and the latency of two loads.
__global__ __launch_bounds__(kWave) void tree_kernel(TreeCall c) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const int off = min(max(c.offsets[b], 0), c.tokens), n = min(max(c.offsets[b + 1], 0), c.tokens) - off;
    const int first = c.lengths[b] - n;
    // Rows of no sequence.
    auto clear = [&](int from, int to) {
        for (int i = from + lane; i < to; i += kWave) {
            c.positions[i] = 0;
            c.near[i] = 0;
            c.above[i] = -1;
        }
    };
    if (b == 0) clear(0, off);
    if (b == c.batch - 1) clear(off + max(n, 0), c.tokens);
    for (int block = 0; block < n; block += kWave) {
        const int i = block + lane;
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
            // Positions of earlier tokens are this wave's own writes.
            c.positions[off + i] = above >= 0 ? c.positions[off + above] + 1 + steps : first + steps;
            c.near[off + i] = word;
            c.above[off + i] = above;
        }
        __threadfence_block();
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
// passes u_0 times the whole sum. Sums and products are in 64 bits: a running sum over
// 100,000 tokens of nearly equal weights passes a border within its own float32 error in a
// hundredth of all calls. Values that are not positive and finite count as 0.
//
// Two kernels. verify_kernel: every workgroup walks down its sequence's tree as far as
// that needs no sum over the vocabulary (chosen drafts: to the end; drawn ones: to the
// first that is turned down), 64 drafts at a time in the lanes of a wave, whose p and q
// are fetched together before the first is looked at; then each of its waves adds up a
// part of what is left. sample_kernel, one workgroup per sequence, goes on from there:
// where more drawn drafts are turned down it adds up the whole vocabulary by itself.


template <class E>
struct Probability;  // the value of an element
template <>
struct Probability<float> {
    static __device__ __forceinline__ float value(float x) { return x; }
};
template <>
struct Probability<uint16_t> {  // bf16
    static __device__ __forceinline__ float value(uint16_t x) { return bf16_to_f32(x); }
};
template <>
struct Probability<_Float16> {
    static __device__ __forceinline__ float value(_Float16 x) { return static_cast<float>(x); }
};

// Not a number, negative, infinite: 0.
__device__ __forceinline__ double weight_of(float x) { return x > 0.f && x < INFINITY ? static_cast<double>(x) : 0.0; }

constexpr int kEach = 8;  // neighbouring tokens of the vocabulary that a lane takes at a time
constexpr int kTimes = kVerifyPart / (kWave * kEach);

template <class E>
__device__ __forceinline__ void read_weights(const E* row, int at, int vocab, double (&w)[kEach]) {
    E x[kEach];
    if (at + kEach <= vocab) {
        __builtin_memcpy(x, row + at, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) x[e] = at + e < vocab ? row[at + e] : E(0);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) w[e] = weight_of(Probability<E>::value(x[e]));
}

// A sequence's new tokens.
struct VerifyUnit {
    int off, n;
};

template <class E>
struct Verifier {
    const VerifyCall& c;
    VerifyUnit u;
    int lane;

    __device__ __forceinline__ const E* target(int place) const {
        return static_cast<const E*>(c.target) + int64_t(u.off + place) * c.target_row;
    }
    __device__ __forceinline__ const E* draft(int place) const {
        return static_cast<const E*>(c.draft) + int64_t(u.off + place) * c.draft_row;
    }
    __device__ __forceinline__ int64_t token(int place) const {
        return c.wide ? static_cast<const int64_t*>(c.tokens)[u.off + place] : static_cast<const int32_t*>(c.tokens)[u.off + place];
    }
    // What is left of p behind the last kept token after `less` drafts.
    __device__ __forceinline__ double rest(double p, double q, int less) const {
        const double* totals = c.totals + u.off;
        for (int i = 0; i < less; ++i) {
            const double r = p - (i == 0 ? 1.0 : totals[i]) * q;
            p = r > 0.0 ? r : 0.0;
        }
        return p;
    }

    // Walks on from s, S = sum, until no child is left (true) or, among drawn drafts, one
    // has been turned down (false; s.less counts it). All 64 lanes alike.
    __device__ bool walk(VerifyState& s, double& sum, bool writes) const {
        for (int window = s.next & ~(kWave - 1); window < u.n; window += kWave) {
            const int place = window + lane;
            const bool there = place < u.n;
            const int parent = there ? c.parents[u.off + place] : -1;
            const int64_t x = there ? token(place) : -1;
            const bool inside = parent >= 0 && parent < place && x >= 0 && x < c.vocab;
            double p = 0.0, uq = there ? static_cast<double>(c.uniforms[u.off + place]) : 0.0, q = 1.0;
            if (inside) p = weight_of(Probability<E>::value(target(parent)[x]));
            if (c.draft) {
                q = inside ? weight_of(Probability<E>::value(draft(parent)[x])) : 0.0;
                uq *= q;
            }
            for (;;) {
                const uint64_t left = __ballot(there && parent == s.last && place >= s.next && place > s.last);
                if (left == 0) break;
                const int at = __builtin_ctzll(left);
                double size = __shfl(p, at);
                const double bar = __shfl(uq, at);
                const int64_t its = __shfl(static_cast<long long>(x), at);
                if (c.draft) {
                    size = rest(size, __shfl(q, at), s.less);
                } else if (s.less > 0) {
                    // Chosen before: nothing is left of it.
                    bool again = __ballot(there && parent == s.last && x == its && lane < at) != 0;
                    for (int before = s.last + 1; before < window && !again; before += kWave) {
                        const int i = before + lane;
                        again = __ballot(i < window && c.parents[u.off + i] == s.last && token(i) == its) != 0;
                    }
                    if (again) size = 0.0;
                }
                s.next = window + at + 1;
                if (bar * sum < size) {
                    s.last = window + at;
                    if (writes && lane == 0) c.path[u.off + s.counts] = s.last;
                    ++s.counts;
                    s.less = 0;
                    sum = 1.0;
                } else {
                    ++s.less;
                    if (c.draft) return false;
                    sum -= size;
                }
            }
        }
        return true;
    }

    // What is left of a part: w[i] of the tokens from first_of(part, i) on.
    __device__ __forceinline__ int first_of(int part, int i) const {
        return part * kVerifyPart + (i * kWave + lane) * kEach;
    }
    __device__ __forceinline__ void left_of(const VerifyState& s, int part, double (&w)[kTimes][kEach]) const {
#pragma unroll
        for (int i = 0; i < kTimes; ++i) read_weights(target(s.last), first_of(part, i), c.vocab, w[i]);
        if (s.less == 0) return;
        if (c.draft) {
            double q[kTimes][kEach];
#pragma unroll
            for (int i = 0; i < kTimes; ++i) read_weights(draft(s.last), first_of(part, i), c.vocab, q[i]);
#pragma unroll
            for (int i = 0; i < kTimes; ++i)
#pragma unroll
                for (int e = 0; e < kEach; ++e) w[i][e] = rest(w[i][e], q[i][e], s.less);
            return;
        }
        for (int window = (s.last + 1) & ~(kWave - 1); window < u.n; window += kWave) {
            const int place = window + lane;
            const bool there = place < u.n && place > s.last && c.parents[u.off + place] == s.last;
            const int64_t x = there ? token(place) : -1;
            for (uint64_t gone = __ballot(there && x >= 0 && x < c.vocab); gone; gone &= gone - 1) {
                const int its = __shfl(static_cast<int>(x), __builtin_ctzll(gone));
#pragma unroll
                for (int i = 0; i < kTimes; ++i)
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        if (its == first_of(part, i) + e) w[i][e] = 0.0;
            }
        }
    }

    // The sum of a part, in all lanes.
    __device__ __forceinline__ double part_sum(const VerifyState& s, int part) const {
        double w[kTimes][kEach], sum = 0.0;
        left_of(s, part, w);
#pragma unroll
        for (int i = 0; i < kTimes; ++i)
#pragma unroll
            for (int e = 0; e < kEach; ++e) sum += w[i][e];
#pragma unroll
        for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m);
        return sum;
    }
};

// x and those of the lanes before.
__device__ __forceinline__ double running_sum(double x, int lane) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
        const double before = __shfl_up(x, m);
        if (lane >= m) x += before;
    }
    return x;
}

__device__ __forceinline__ VerifyUnit verify_unit(const VerifyCall& c, int b) {
    const int off = min(max(c.offsets[b], 0), c.rows);
    return {off, min(max(c.offsets[b + 1], 0), c.rows) - off};
}

template <class E>
__global__ __launch_bounds__(256) void verify_kernel(VerifyCall c) {
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Verifier<E> v{c, verify_unit(c, b), lane};
    if (v.u.n <= 0) return;
    const bool writes = blockIdx.x == 0 && wave == 0;
    VerifyState s{0, 1, 1, 0};
    double sum = 1.0;
    v.walk(s, sum, writes);
    if (writes && lane == 0) c.state[b] = s;
    const int part = blockIdx.x * 4 + wave;
    if (part >= c.parts) return;
    const double total = v.part_sum(s, part);
    if (lane == 0) c.sums[int64_t(b) * c.parts + part] = total;
}

constexpr int kSampleWaves = 16;

template <class E>
__global__ __launch_bounds__(kSampleWaves * kWave) void sample_kernel(VerifyCall c) {
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Verifier<E> v{c, verify_unit(c, b), lane};
    const VerifyUnit u = v.u;
    // Rows of no sequence have no path.
    if (b == 0)
        for (int i = threadIdx.x; i < u.off; i += blockDim.x) c.path[i] = -1;
    if (b == c.batch - 1)
        for (int i = u.off + max(u.n, 0) + threadIdx.x; i < c.rows; i += blockDim.x) c.path[i] = -1;
    auto finish = [&](int counts, int64_t next) {
        c.counts[b] = counts;
        if (c.wide) static_cast<int64_t*>(c.next)[b] = next;
        else static_cast<int32_t*>(c.next)[b] = static_cast<int32_t>(next);
    };
    if (u.n <= 0) {
        if (threadIdx.x == 0) finish(0, -1);
        return;
    }
    double* sums = c.sums + int64_t(b) * c.parts;
    double* totals = c.totals + u.off;
    VerifyState s = c.state[b];
    auto whole = [&]() {  // the sum of all parts, in order, in all lanes
        double sum = 0.0;
        for (int p = 0; p < c.parts; p += kWave) {
            const double run = running_sum(p + lane < c.parts ? sums[p + lane] : 0.0, lane);
            sum += __shfl(run, kWave - 1);
        }
        return sum;
    };
    auto add_up = [&]() {
        __syncthreads();  // every wave is done with the sums before
        for (int p = wave; p < c.parts; p += kSampleWaves) {
            const double sum = v.part_sum(s, p);
            if (lane == 0) sums[p] = sum;
        }
        __threadfence_block();
        __syncthreads();
    };
    double sum = whole();
    if (c.draft) {
        bool walked = s.less == 0;
        while (!walked) {
            // The sums are of what the draft that was turned down last has left.
            bool stale = false;
            if (sum > 0.0) {
                if (threadIdx.x == 0) totals[s.less] = sum;
                __threadfence_block();
                __syncthreads();
            } else {  // nothing is left: it changes nothing
                --s.less;
                sum = s.less == 0 ? 1.0 : totals[s.less];
                stale = true;
            }
            const int counts = s.counts, less = s.less;
            walked = v.walk(s, sum, wave == 0);
            if (stale || s.counts != counts || s.less != less) {
                add_up();
                sum = whole();
            }
        }
    }
    // The next token.
    for (int i = s.counts + threadIdx.x; i < u.n; i += blockDim.x) c.path[u.off + i] = -1;
    if (wave != 0) return;
    if (lane == 0) c.path[u.off] = 0;
    const double border = static_cast<double>(c.uniforms[u.off]) * sum;
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
            base = before + (at > 0 ? __shfl(run, at - 1) : 0.0);
        }
        before += __shfl(run, kWave - 1);
    }
    int found = -1;  // the token in it, likewise
    if (part >= 0) {
        double w[kTimes][kEach];
        v.left_of(s, part, w);
        past = false;
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
                found = __shfl(v.first_of(part, i) + (past ? first : any), past ? __builtin_ctzll(passes) : 63 - __builtin_clzll(has));
            }
            base += __shfl(run, kWave - 1);
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
    hipLaunchKernelGGL(tree_kernel, dim3(static_cast<unsigned>(c.batch)), dim3(kWave), 0, stream, c);
    return check_launch("tree_kernel");
}

int launch_verify(const VerifyCall& c, hipStream_t stream) {
    return c.type == 0 ? launch_verify_as<uint16_t>(c, stream)
         : c.type == 1 ? launch_verify_as<_Float16>(c, stream) : launch_verify_as<float>(c, stream);
}

}  // namespace ab
