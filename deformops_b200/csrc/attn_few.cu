// Cross attention forward for at most 16 rows to a key head: one new token of a sequence and the like.
//
// Bound by reading k and v once.  They go straight from memory to the registers of matrix instructions, 16 bytes to
// a lane, without shared memory: a product's inner index may run in any order, and so may the columns of its result.
//
//   scores   B = k: the lanes t = 0 .. 3 of a state have its channels 8 t .. 8 t + 7 of every 32, in inner order
//            (2 t, 2 t + 1, 2 t + 8, 2 t + 9) of two products; q lies in the same order
//   O        B = v: lane (g, t) has channels 8 g .. 8 g + 7 of states 2 t, 2 t + 1, 2 t + 8 and 2 t + 9, two states
//            packed to a register; column g of product i is channel 8 g + i
//
// With at most eight rows (EIGHT) the second product is O^T = v^T p^T, the channels 8 g + 2 i and 8 g + 2 i + 1 as
// rows g and g + 8 of product i: half the products and half the registers for O, so more warps.
//
// (float32: four channels to 16 bytes, two terms of tf32, products of 8 instead of 16.  What is left out is 2^-21 of a
// product, eight times as much as by the kernels of many rows: third terms would double the products.
// 16 bits: weights are rounded to the type, as there.)  Every warp takes blocks
// of its CTA's stretch of states with a running maximum and sum of its own; the warps, and the stretches
// (attn_aux.cu), are joined at the end.
//
// bf16: 512 caches of 4000 states of 64 channels 89 us (5.9 TB/s), 512 of 8000 of 128 340 us (6.2 TB/s), 128 of 1500 of 128
// 23 us (4.2 TB/s, and 3 to join three parts).  float32: 216 us (4.9 TB/s), 1226 (3.4 TB/s) and 76 in all.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "warp_mma.cuh"

namespace msda_b200 {

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;

// states of a block: 4 KB of k and v to a warp at a time and more, as far as registers go
template <typename T, int DP>
constexpr int kBlock = sizeof(T) == 4 ? (DP == 128 ? 8 : 16) : DP == 32 ? 32 : 16;

// CTAs to an SM, as registers allow
template <typename T, int DP, bool EIGHT>
constexpr int kResident = DP == 128 ? (EIGHT && sizeof(T) == 2 ? 3 : 2) : sizeof(T) == 4 && DP == 64 ? (EIGHT ? 4 : 3) : EIGHT ? 5 : 4;

template <typename T, int DP>
struct Few {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int KB = kBlock<T, DP>, NT = KB / 8;         // states, and score products of 8 of them
    static constexpr int kInner = kWide ? 16 : 32, KC = DP / kInner;        // channels of a state's four lanes
    // channels of a lane of v, and of all of them; a thread has kLane 32-bit registers of one state
    static constexpr int kChannels = kWide ? 4 : DP == 32 ? 4 : 8, kSpan = 8 * kChannels, VC = DP / kSpan;
    static constexpr int kLane = kWide ? 4 : kChannels / 2;
    static constexpr int kStates = KB / 4;                        // states of v of a thread
};

template <int N>
__device__ __forceinline__ void load_lane(uint32_t (&r)[N], const void *p, bool valid) {
    if constexpr (N == 4) {
        const uint4 x = valid ? ldg16(p) : make_uint4(0, 0, 0, 0);
        r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
    } else {
        const uint2 x = valid ? __ldg(static_cast<const uint2 *>(p)) : make_uint2(0, 0);
        r[0] = x.x, r[1] = x.y;
    }
}

template <typename T, int DP, bool EIGHT>
__global__ void __launch_bounds__(kThreads, kResident<T, DP, EIGHT>) attention_few_kernel(const __grid_constant__ AttentionParams p) {
    using F = Few<T, DP>;
    constexpr int KB = F::KB, NT = F::NT, KC = F::KC, VC = F::VC, CH = F::kChannels;
    __shared__ float s_max[kWarps][16], s_sum[kWarps][16];
    extern __shared__ float s_out[];                               // (warps, rows, DP)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    grid_launch_dependents();
    grid_dependency_wait();            // (of the masks that this call has packed)
    const unsigned bh = blockIdx.x / p.splits;
    const int part = (int)(blockIdx.x - bh * p.splits), b = (int)(bh / p.K), h = (int)(bh - b * p.K);
    const T *k = static_cast<const T *>(p.k) + b * p.ks[0] + h * p.ks[2];
    const T *v = static_cast<const T *>(p.v) + b * p.vs[0] + h * p.vs[2];
    const uint32_t *words = key_words_of(p, b, h);
    constexpr int kHalves = EIGHT ? 1 : 2;                         // rows g, and g + 8
    // float16: exponent of what the weights, 1 at most, are multiplied by, and their sum with them (small ones keep their bits)
    constexpr float kUp = kScaled<T> ? 15.f : 0.f;
    constexpr int CO = EIGHT ? CH / 2 : CH;                        // products of a span of channels

    uint32_t q[kHalves][KC][4];
    const uint32_t *rw[kHalves];
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
        const int r = g + 8 * half;
        const T *from = static_cast<const T *>(p.q) + (r < p.R ? row_offset(p.qs, p.share, b, h, r) : 0);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int d = c * F::kInner + t * (F::kInner / 4);
            load_lane(q[half][c], from + d, r < p.R && d < p.D);
        }
        rw[half] = r < p.R ? row_words_of(p, b, h, r) : nullptr;
    }

    float o[VC][CO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int i = 0; i < CO; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;

    const int end = (int)min((int64_t)p.S, (int64_t)(part + 1) * p.tiles * KB);
    for (int first = part * p.tiles * KB + warp * KB; first < end; first += kWarps * KB) {
        // bit i: state first + i may be seen by somebody
        const uint32_t seen = (key_word(words, p.S, first >> 5) >> (first & 31)) & (KB == 32 ? 0xffffffffu : (1u << KB) - 1);
        if (seen == 0) continue;
        uint32_t fk[NT][KC][4], fv[F::kStates][VC][F::kLane];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int i = n * 8 + g, d = c * F::kInner + t * (F::kInner / 4);
                load_lane(fk[n][c], k + (first + i) * p.ks[1] + d, ((seen >> i) & 1) && d < p.D);
            }
#pragma unroll
        for (int n = 0; n < F::kStates; ++n)
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                const int i = (n >> 1) * 8 + 2 * t + (n & 1), d = c * F::kSpan + g * CH;
                load_lane(fv[n][c], v + (first + i) * p.vs[1] + d, ((seen >> i) & 1) && d < p.D);
            }
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const uint32_t a[4] = {q[0][c][i], EIGHT ? 0u : q[kHalves - 1][c][i], q[0][c][i + 1], EIGHT ? 0u : q[kHalves - 1][c][i + 1]};
                    if constexpr (F::kWide) {
                        uint32_t ah[4], al[4], bh2[2], bl[2];
#pragma unroll
                        for (int j = 0; j < 4; ++j) split_tf32(__uint_as_float(a[j]), ah[j], al[j]);
                        split_tf32(__uint_as_float(fk[n][c][i]), bh2[0], bl[0]);
                        split_tf32(__uint_as_float(fk[n][c][i + 1]), bh2[1], bl[1]);
                        mma_tf32x3(s[n], ah, al, bh2, bl);
                    } else {
                        mma16<T>(s[n], a, fk[n][c][i], fk[n][c][i + 1]);
                    }
                }
        }
        float keep[2] = {1.f, 1.f};
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
            uint32_t bits = seen;
            if (rw[half] != nullptr) bits = __ldg(rw[half] + (first >> 5)) >> (first & 31);
            float top = m[half];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float &x = s[n][2 * half + e];
                    x = (bits >> (n * 8 + 2 * t + e)) & 1 ? x * p.scale_log2 : -INFINITY;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float base = top == -INFINITY ? 0.f : top;           // nothing seen so far
            keep[half] = fast_exp2(m[half] - base);
            m[half] = top;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][2 * half + e] = fast_exp2(s[n][2 * half + e] - base + kUp);       // (less than base first: exact)
                    sum += s[n][2 * half + e];
                }
            l[half] = l[half] * keep[half] + sum;
        }
        if constexpr (EIGHT) {
            // (the lanes of row r are 4 r .. 4 r + 3; O has rows 2 t and 2 t + 1 here)
            const float mine = keep[0];
            keep[0] = __shfl_sync(0xffffffffu, mine, 8 * t), keep[1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
        }
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int i = 0; i < CO; ++i) {
                if constexpr (F::kWide) {
                    // (from zero, and added with rounding: a matrix instruction cuts its sums off)
                    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t ah[4], al[4], bh2[2], bl[2];
                        if constexpr (EIGHT) {
                            split_tf32(__uint_as_float(fv[2 * n][c][2 * i]), ah[0], al[0]);
                            split_tf32(__uint_as_float(fv[2 * n][c][2 * i + 1]), ah[1], al[1]);
                            split_tf32(__uint_as_float(fv[2 * n + 1][c][2 * i]), ah[2], al[2]);
                            split_tf32(__uint_as_float(fv[2 * n + 1][c][2 * i + 1]), ah[3], al[3]);
                            split_tf32(s[n][0], bh2[0], bl[0]), split_tf32(s[n][1], bh2[1], bl[1]);
                        } else {
                            split_tf32(s[n][0], ah[0], al[0]), split_tf32(s[n][2], ah[1], al[1]);
                            split_tf32(s[n][1], ah[2], al[2]), split_tf32(s[n][3], ah[3], al[3]);
                            split_tf32(__uint_as_float(fv[2 * n][c][i]), bh2[0], bl[0]);
                            split_tf32(__uint_as_float(fv[2 * n + 1][c][i]), bh2[1], bl[1]);
                        }
                        mma_tf32x3(add, ah, al, bh2, bl);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][i][e] = fmaf(o[c][i][e], keep[EIGHT ? e & 1 : e >> 1], add[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][i][e] *= keep[EIGHT ? e & 1 : e >> 1];
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        // a channel of two neighbouring states: the lower or the upper halves of two registers
                        const auto pair = [&](int state, int channel) {
                            return __byte_perm(fv[state][c][channel >> 1], fv[state + 1][c][channel >> 1], channel & 1 ? 0x7632 : 0x5410);
                        };
                        if constexpr (EIGHT) {
                            const uint32_t a[4] = {pair(2 * n, 2 * i), pair(2 * n, 2 * i + 1), pair(2 * n + 2, 2 * i), pair(2 * n + 2, 2 * i + 1)};
                            mma16<T>(o[c][i], a, VecTraits<T>::pack2(make_float2(s[n][0], s[n][1])),
                                     VecTraits<T>::pack2(make_float2(s[n + 1][0], s[n + 1][1])));
                        } else {
                            const uint32_t a[4] = {VecTraits<T>::pack2(make_float2(s[n][0], s[n][1])),
                                                   VecTraits<T>::pack2(make_float2(s[n][2], s[n][3])),
                                                   VecTraits<T>::pack2(make_float2(s[n + 1][0], s[n + 1][1])),
                                                   VecTraits<T>::pack2(make_float2(s[n + 1][2], s[n + 1][3]))};
                            mma16<T>(o[c][i], a, pair(2 * n, i), pair(2 * n + 2, i));
                        }
                    }
                }
            }
    }

    // the warps' parts: a thread to a channel of a row
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
        const int r = g + 8 * half;
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        if (t == 0 && r < p.R) s_max[warp][r] = m[half], s_sum[warp][r] = l[half];
    }
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int i = 0; i < CO; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = EIGHT ? 2 * t + (e & 1) : g + 8 * (e >> 1);
                const int d = c * F::kSpan + (EIGHT ? g * CH + 2 * i + (e >> 1) : (2 * t + (e & 1)) * CH + i);
                if (r < p.R) s_out[(warp * p.R + r) * DP + d] = o[c][i][e];
            }
    __syncthreads();
    const int64_t rows = (int64_t)p.B * p.K * p.R;
    for (int i = threadIdx.x; i < p.R * p.D; i += kThreads) {
        const int r = i / p.D, d = i - r * p.D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_max[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
        float total = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float weight = fast_exp2(s_max[w][r] - base);
            total += weight * s_sum[w][r];
            x += weight * s_out[(w * p.R + r) * DP + d];
        }
        x = total == 0.f ? 0.f : x / total;
        const float lse = total == 0.f ? (p.splits > 1 ? -INFINITY : INFINITY) : top - kUp + log2f(total);
        const int64_t at = (int64_t)bh * p.R + r;
        const int query = r / p.share;
        if (p.splits > 1) {
            p.part[(part * rows + at) * p.D + d] = x;
            if (d == 0) p.part_lse[part * rows + at] = lse;
        } else {
            static_cast<T *>(p.out)[(((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (r - query * p.share)) * p.D + d] =
                VecTraits<T>::from_float(x);
            if (d == 0) p.lse[at] = lse;
        }
    }
}

template <typename T, int DP, bool EIGHT>
cudaError_t launch_rows(const AttentionParams &p, cudaStream_t stream) {
    const auto kernel = attention_few_kernel<T, DP, EIGHT>;
    constexpr int most = kWarps * (EIGHT ? 8 : 16) * DP * sizeof(float);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)p.B * p.K * p.splits;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, dim3((unsigned)grid), kThreads, kWarps * p.R * DP * sizeof(float), stream, p);
}

template <typename T, int DP>
cudaError_t launch(const AttentionParams &p, cudaStream_t stream) {
    return p.R <= 8 ? launch_rows<T, DP, true>(p, stream) : launch_rows<T, DP, false>(p, stream);
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, cudaStream_t stream) {
    return p.D <= 32 ? launch<T, 32>(p, stream) : p.D <= 64 ? launch<T, 64>(p, stream) : launch<T, 128>(p, stream);
}

template <typename T, int DP>
FewShape shape(int64_t rows) {
    return {kBlock<T, DP>, rows <= 8 ? kResident<T, DP, true> : kResident<T, DP, false>};
}
template <typename T>
FewShape shape_typed(int64_t D, int64_t rows) {
    return D <= 32 ? shape<T, 32>(rows) : D <= 64 ? shape<T, 64>(rows) : shape<T, 128>(rows);
}

}  // namespace

FewShape attention_few_shape(int dtype, int64_t D, int64_t rows) {
    return dtype == 0 ? shape_typed<float>(D, rows) : shape_typed<__half>(D, rows);
}

cudaError_t launch_attention_few(const AttentionParams &p, int dtype, cudaStream_t stream) {
    return dtype == 0 ? launch_typed<float>(p, stream)
           : dtype == 1 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream);
}

}  // namespace msda_b200
