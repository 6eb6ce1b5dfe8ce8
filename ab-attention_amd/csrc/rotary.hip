// Rotary positions over several axes (time, height, width).
//
// A pair (x, y) of a row's values turns by the angle p f of its axis' position p
// and its frequency f = theta^(-2j / d) (j-th pair of an axis of d dims; joint:
// of all axes' dims together):
//   x' = x cos - y sin,  y' = x sin + y cos.
// The gradient is the rotation by the opposite angle. Angles are reduced to a
// fraction of a turn in 64 bits (positions of 10^5 and more keep their last
// bits), their sine and cosine taken in float32, and each result is rounded to
// its type once. Every thread holds the sines of one token's few pairs and
// walks over heads of Q, then of K, so that their cost (some 250 instructions) is
// shared by the heads. What bounds the kernel is reading and writing the rows: Q and K
// of 2 x 12 heads x 32,760 tokens in bf16 157 us, 5.1 TB/s (a copy reaches 4.9); a
// token of 8 sequences 6.5 us, its chain of loads and sines.
#include <algorithm>

#include "rotary.hpp"

namespace ab {
namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;  // values of a row that a thread takes at once

// Eight values of a type as floats, from and to 16-byte aligned memory.
template <class T>
struct Values {
    static __device__ __forceinline__ void load(const void* p, float (&x)[kUnit]) {
        const u32x4 w = *static_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = T::lo(w[i]);
            x[2 * i + 1] = T::hi(w[i]);
        }
    }
    static __device__ __forceinline__ void store(void* p, const float (&x)[kUnit]) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = T::pack(x[2 * i], x[2 * i + 1]);
        *static_cast<u32x4*>(p) = w;
    }
    static constexpr int kBytes = 2;
};
struct F32 {};
template <>
struct Values<F32> {
    static __device__ __forceinline__ void load(const void* p, float (&x)[kUnit]) {
        const f32x4 a = static_cast<const f32x4*>(p)[0], b = static_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    }
    static __device__ __forceinline__ void store(void* p, const float (&x)[kUnit]) {
        static_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
        static_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
    static constexpr int kBytes = 4;
};

// Sines and cosines of kPairs pairs from `first` on at a token's positions, those at
// `end` and behind it left as they are. The frequency of the first one is an
// exponential; its neighbours' follow by the axis' ratio, a rounding of 2^-53 each.
template <int kPairs>
__device__ __forceinline__ void turns(const RotaryCall& c, int64_t token, int first, int end, float (&s)[kPairs], float (&co)[kPairs]) {
    int axis = 0, begin = 0;  // the first pair's axis, and that axis' first pair
#pragma unroll
    for (int a = 0; a < kMaxAxes - 1; ++a) {
        const int pairs = c.pairs[a];
        if (axis == a && a < c.axes - 1 && first - begin >= pairs) {
            ++axis;
            begin += pairs;
        }
    }
    auto position = [&](int a) {
        const int64_t at = token * c.axes + a;
        return c.position_kind == 0   ? static_cast<double>(static_cast<const int32_t*>(c.positions)[at])
               : c.position_kind == 1 ? static_cast<double>(static_cast<const int64_t*>(c.positions)[at])
                                      : static_cast<double>(static_cast<const float*>(c.positions)[at]);
    };
    double p = position(axis) * 0.15915494309189533577;  // 1 / (2 pi): turns at frequency 1
    double frequency = exp2(-(c.joint ? c.step[0] * first : c.step[axis] * (first - begin)));
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        if (first + i >= end) break;
        if (i > 0) {
            if (axis < c.axes - 1 && first + i - begin >= c.pairs[axis]) {
                begin += c.pairs[axis];
                p = position(++axis) * 0.15915494309189533577;
                frequency = c.joint ? frequency * c.ratio[0] : 1.0;
            } else {
                frequency *= c.ratio[c.joint ? 0 : axis];
            }
        }
        const double turns = p * frequency;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s[i], &co[i]);
        s[i] *= c.sign;
    }
}

// Thread: one unit of one token. Adjacent pairs: eight values, four pairs.
// Halves: eight values of the first half and the eight that they pair with.
template <class T, bool kHalves>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryCall c) {
    using V = Values<T>;
    touch(c.in[0], c.out_rows[0].token, c.positions, c.heads[0], c.units, c.per_batch);
    const uint32_t g = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t units = c.units;
    const uint32_t token = g / units, unit = g - token * units;  // token of all batch items
    if (token >= c.total) return;
    const uint32_t b = token / c.tokens, t = token - b * c.tokens;
    const int half = c.turned / 2;
    // Values from `at` on; units behind the turned dims are copied.
    const bool copied = kHalves ? static_cast<int>(unit) * kUnit >= half : static_cast<int>(unit) * kUnit >= c.turned;
    const int at = kHalves && copied ? c.turned + (unit * kUnit - half) : unit * kUnit;

    // Heads of Q and K as one list; this workgroup's are from `head0` on. kAhead rows
    // are read before the first is written, the first ones before the sines are made.
    const int heads = c.heads[0] + c.heads[1];
    const int head0 = blockIdx.y * c.heads_each, head1 = min(head0 + c.heads_each, heads);
    auto place = [&](const Rows& r, int tensor, int h) {
        return (b * r.batch + (h - (tensor ? c.heads[0] : 0)) * r.head + t * r.token + at) * V::kBytes;
    };
    constexpr int kAhead = 4;
    float x[kAhead][kUnit], y[kHalves ? kAhead : 1][kUnit];
    auto read = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = min(h0 + i, head1 - 1), k = h >= c.heads[0];
            const char* src = static_cast<const char*>(c.in[k]) + place(c.in_rows[k], k, h);
            V::load(src, x[i]);
            if constexpr (kHalves)
                if (!copied) V::load(src + half * V::kBytes, y[i]);
        }
    };
    read(head0);

    constexpr int kPairs = kHalves ? 8 : 4;
    float s[kPairs] = {}, co[kPairs] = {};
    if (!copied) turns<kPairs>(c, c.per_batch ? token : t, kHalves ? at : at / 2, half, s, co);

    for (int h0 = head0; h0 < head1; h0 += kAhead) {
        if (h0 > head0) read(h0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = h0 + i, k = h >= c.heads[0];
            if (h >= head1) break;
            char* dst = static_cast<char*>(c.out[k]) + place(c.out_rows[k], k, h);
            if (copied) {
                V::store(dst, x[i]);
                continue;
            }
            if constexpr (kHalves) {
                float u[kUnit], w[kUnit];
#pragma unroll
                for (int e = 0; e < kUnit; ++e) {
                    u[e] = __builtin_fmaf(-y[i][e], s[e], x[i][e] * co[e]);
                    w[e] = __builtin_fmaf(x[i][e], s[e], y[i][e] * co[e]);
                }
                V::store(dst, u);
                V::store(dst + half * V::kBytes, w);
            } else {
                // A unit may hold the last turned pairs and the first copied ones.
                float u[kUnit];
#pragma unroll
                for (int e = 0; e < kPairs; ++e) {
                    const bool turned = at / 2 + e < half;
                    const float p = x[i][2 * e], q = x[i][2 * e + 1];
                    u[2 * e] = turned ? __builtin_fmaf(-q, s[e], p * co[e]) : p;
                    u[2 * e + 1] = turned ? __builtin_fmaf(p, s[e], q * co[e]) : q;
                }
                V::store(dst, u);
            }
        }
    }
}
}  // namespace

int launch_rotary(const RotaryCall& call, int dtype, bool halves, hipStream_t stream) {
    RotaryCall c = call;
    const int64_t threads = int64_t(c.total) * c.units, heads = c.heads[0] + c.heads[1];
    const int64_t blocks = (threads + kThreads - 1) / kThreads;
    // Heads of a thread: all of them, or fewer where that would leave the chip
    // without eight workgroups per CU.
    const int64_t splits = std::clamp<int64_t>(2048 / std::max<int64_t>(blocks, 1), 1, (heads + 3) / 4);
    c.heads_each = static_cast<int32_t>((heads + splits - 1) / splits);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + c.heads_each - 1) / c.heads_each));
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, c);
        return check_launch("rotary_kernel");
    };
    if (dtype == 0) return halves ? run(rotary_kernel<Bf16, true>) : run(rotary_kernel<Bf16, false>);
    if (dtype == 1) return halves ? run(rotary_kernel<F16, true>) : run(rotary_kernel<F16, false>);
    return halves ? run(rotary_kernel<F32, true>) : run(rotary_kernel<F32, false>);
}

}  // namespace ab
