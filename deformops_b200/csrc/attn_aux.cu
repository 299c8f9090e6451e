// Cross attention: masks to bits, rowsum(do o), and the joining of split passes.  All of them read
// their input once and are bound by that, or by their launch: 4 to 6 us each for 4 x 17 821 states and 4 x 300 queries of 8
// heads of 32 (dependent launches hide half of it); the terms of k and v of two such samples 27 us for 182 MB; float16, with
// norms of v's rows, rowsum(do o) of 8 x 100 queries over 4096 states 9 us where it was 5, the bounds 6, most of them under way with it.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"

namespace msda_b200 {

namespace {

constexpr int kThreads = 256;

// Lists of a sample's tiles, by one CTA: positions by counting within warps, then over the warps.
template <int BN>
__device__ void list_tiles(const uint32_t *words, int S, uint32_t *count, uint32_t *list) {
    __shared__ int warps[33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tiles = (S + BN - 1) / BN;
    int done = 0;
    for (int base = 0; base < tiles; base += 1024) {
        const int tile = base + threadIdx.x;
        uint32_t any = 0, all = 0xffffffffu;
        if (tile < tiles)
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
                const uint32_t w = words[tile * (BN / 32) + i];
                any |= w, all &= w;
            }
        const uint32_t mine = __ballot_sync(0xffffffffu, any != 0);
        if (lane == 0) warps[warp] = __popc(mine);
        __syncthreads();
        if (warp == 0) {
            int n = warps[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int from = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += from;
            }
            warps[lane + 1] = n;
        }
        __syncthreads();
        const int before = warp == 0 ? 0 : warps[warp];
        if (any != 0)
            list[done + before + __popc(mine & ((1u << lane) - 1))] = (uint32_t)tile | (all == 0xffffffffu ? 0x80000000u : 0u);
        done += warps[32];
        __syncthreads();
    }
    if (threadIdx.x == 0) *count = done;
}
__device__ void list_both(const uint32_t *words, int S, uint32_t *lists) {
    list_tiles<64>(words, S, lists, lists + 2);
    list_tiles<128>(words, S, lists + 1, lists + 2 + (S + 63) / 64);
}

// 32 states' bits, a lane to a state; nothing before `S`
__device__ __forceinline__ uint32_t pack_word(const uint8_t *hidden, int64_t stride, int state, int S) {
    return __ballot_sync(0xffffffffu, state < S && __ldg(hidden + state * stride) == 0);
}

// Words first .. first + 31 of a mask row, one to a lane.  States that are neighbours are read 16 bytes to a lane from
// the last 16-byte boundary on, and the bytes that were asked for are moved into place on the way (rows of odd
// length have no alignment); others a byte to a lane.
__device__ __forceinline__ uint32_t pack_words(const uint8_t *hidden, int64_t stride, int first, int W, int S) {
    const int lane = threadIdx.x & 31;
    uint32_t word = 0;
    if (stride != 1) {
        for (int i = 0; i < 32 && first + i < W; ++i) {
            const uint32_t x = pack_word(hidden, stride, (first + i) * 32 + lane, S);
            if (i == lane) word = x;
        }
        return word;
    }
    // lane i: the bytes of 32 states, from three aligned vectors
    const int state = (first + lane) * 32, left = S - state;
    const uintptr_t at = reinterpret_cast<uintptr_t>(hidden + state);
    const uint4 *from = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15);
    const int off = (int)(at & 15);
    uint32_t bits[2] = {0, 0};
#pragma unroll
    for (int v = 0; v < 3; ++v) {
        // (a vector with one byte that exists lies within the allocation's 16-byte granule)
        if (left > 0 && 16 * v - off < min(left, 32)) {
            const uint4 x = __ldg(from + v);
            const uint32_t in[4] = {x.x, x.y, x.z, x.w};
            uint32_t seen = 0;                                               // of 16 bytes
#pragma unroll
            for (int i = 0; i < 4; ++i)
                // each byte 0 or not: its lowest bit to bit 4 i + byte
                seen |= ((__vcmpeq4(in[i], 0) & 0x08040201u) * 0x01010101u >> 24) << (4 * i);
            if (v < 2)
                bits[0] |= seen << (16 * v);
            else
                bits[1] = seen;
        }
    }
    word = __funnelshift_r(bits[0], bits[1], off);
    return left >= 32 ? word : left <= 0 ? 0u : word & ((1u << left) - 1);
}

// padding alone: a CTA to a sample packs it and lists its tiles
__global__ void __launch_bounds__(1024) attention_padding_kernel(const __grid_constant__ MaskParams p) {
    grid_launch_dependents();
    const int lane = threadIdx.x & 31, b = blockIdx.x;
    uint32_t *words = p.key_words + (int64_t)b * p.W;
    for (int first = threadIdx.x & ~31; first < p.W; first += 1024) {
        const uint32_t word = pack_words(p.padding + b * p.ps[0], p.ps[1], first, p.W, p.S);
        if (first + lane < p.W) words[first + lane] = word;
    }
    __syncthreads();
    list_both(words, p.S, p.lists + b * list_words(p.S));
}

// a warp to 1024 states of a mask row at a time
__global__ void __launch_bounds__(kThreads) attention_mask_kernel(const __grid_constant__ MaskParams p) {
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int groups = (p.W + 31) / 32;
    const int64_t rows = (int64_t)p.B * p.H * p.Q, tasks = rows * groups;
    for (int64_t task = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); task < tasks;
         task += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t row = task / groups;
        const int first = (int)(task - row * groups) * 32;                 // word
        const int64_t bh = row / p.Q, query = row - bh * p.Q, b = bh / p.H;
        uint32_t word = pack_words(p.mask + b * p.ms[0] + (bh - b * p.H) * p.ms[1] + query * p.ms[2], p.ms[3], first, p.W, p.S);
        if (p.padding != nullptr) word &= pack_words(p.padding + b * p.ps[0], p.ps[1], first, p.W, p.S);
        if (first + lane < p.W) p.row_words[row * p.W + first + lane] = word;
    }
}

// key words: the or of all rows of a sample (or of the heads that share a key head)
__global__ void __launch_bounds__(1024) attention_mask_any_kernel(const __grid_constant__ MaskParams p) {
    __shared__ uint32_t any[32][33];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int blocks = (p.W + 31) / 32;
    const int bk = blockIdx.x / blocks, w = (blockIdx.x - bk * blocks) * 32 + lane;
    const int64_t rows = (int64_t)(p.H / p.KW) * p.Q;              // consecutive ones
    uint32_t found = 0;
    if (w < p.W)
        for (int64_t r = part; r < rows; r += 32) found |= p.row_words[(bk * rows + r) * p.W + w];
    any[part][lane] = found;
    __syncthreads();
    found = __reduce_or_sync(0xffffffffu, any[lane][part]);
    const int word = (blockIdx.x - bk * blocks) * 32 + part;
    if (lane == 0 && word < p.W) p.key_words[(int64_t)bk * p.W + word] = found;
}

__global__ void __launch_bounds__(1024) attention_list_kernel(const __grid_constant__ MaskParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    list_both(p.key_words + (int64_t)blockIdx.x * p.W, p.S, p.lists + blockIdx.x * list_words(p.S));
}

// a thread to eight channels, zeros behind the last one; blockIdx.y: the tensor
__global__ void __launch_bounds__(kThreads) attention_terms_kernel(const __grid_constant__ TermsParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const TermsParams::Tensor &t = p.of[blockIdx.y];
    const unsigned chunks = (p.D + 7) / 8;
    const int64_t all = (int64_t)p.B * t.tokens * t.heads * chunks;
    uint4 *terms = static_cast<uint4 *>(t.terms);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / chunks, token = row / t.heads, b = token / t.tokens;
        const int c = (int)(i - row * chunks) * 8;
        const float *from = static_cast<const float *>(t.x) + b * t.strides[0] + (token - b * t.tokens) * t.strides[1] +
                            (row - token * t.heads) * t.strides[2] + c;
        const float4 lo = __ldg(reinterpret_cast<const float4 *>(from));
        const float4 hi = c + 4 < p.D ? __ldg(reinterpret_cast<const float4 *>(from + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
        uint32_t w[4][3];
        split_terms(make_float2(lo.x, lo.y), w[0]), split_terms(make_float2(lo.z, lo.w), w[1]);
        split_terms(make_float2(hi.x, hi.y), w[2]), split_terms(make_float2(hi.z, hi.w), w[3]);
#pragma unroll
        for (int k = 0; k < 3; ++k) terms[k * all + i] = make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]);
    }
}

constexpr int kRowsAtOnce = 4, kDeltaRows = kThreads / 8 * kRowsAtOnce;

// Norms of v's rows, LANES lanes to one, rows in the order of dense states, a CTA to kStateRows of a sample.  What unseen
// states hold is read with the rest, so as not to wait for the mask, and not used.
template <int LANES>
constexpr int kStateRows = kThreads / LANES * kRowsAtOnce;
template <typename T, int LANES>
__device__ __forceinline__ void state_norms(const AttentionParams &p, unsigned block) {
    constexpr int kVec = VecTraits<T>::kVec, kStep = kThreads / LANES;
    const int64_t all = (int64_t)p.S * p.K;
    const unsigned blocks = (unsigned)((all + kStateRows<LANES> - 1) / kStateRows<LANES>);
    const int b = (int)(block / blocks), lane = threadIdx.x & (LANES - 1);
    const int64_t row = (int64_t)(block - b * blocks) * kStateRows<LANES> + threadIdx.x / LANES;
    int state = all >> 32 != 0 ? (int)(row / p.K) : (int)((unsigned)row / p.K), h = (int)(row - (int64_t)state * p.K);
    const int states = kStep / p.K, heads = kStep - states * p.K;
    uint4 x[kRowsAtOnce];
    float sum[kRowsAtOnce] = {};
    int64_t at[kRowsAtOnce];
    const T *from[kRowsAtOnce];
    bool seen[kRowsAtOnce];
#pragma unroll
    for (int k = 0; k < kRowsAtOnce; ++k) {
        const bool there = row + k * kStep < all;
        at[k] = there ? ((int64_t)b * p.K + h) * p.S + state : -1;
        from[k] = there ? static_cast<const T *>(p.v) + b * p.vs[0] + state * p.vs[1] + h * p.vs[2] : nullptr;
        seen[k] = there && ((key_word(key_words_of(p, b, h), p.S, state >> 5) >> (state & 31)) & 1);
        state += states, h += heads;
        if (h >= p.K) h -= p.K, ++state;
    }
    for (int c = lane * kVec; c < p.D; c += LANES * kVec) {
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) x[k] = from[k] != nullptr ? ldg16(from[k] + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            float2 u[kVec / 2];
            VecTraits<T>::unpack(x[k], u);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) sum[k] += u[i].x * u[i].x + u[i].y * u[i].y;
        }
    }
#pragma unroll
    for (int k = 0; k < kRowsAtOnce; ++k) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
        if (lane == 0 && at[k] >= 0) p.state_norms[at[k]] = seen[k] ? sqrtf(sum[k]) : 0.f;
    }
}

// eight lanes to a row, rows in the order of `out`; float16: CTAs behind the last row take v's
template <typename T>
__global__ void __launch_bounds__(kThreads) attention_delta_kernel(const __grid_constant__ AttentionParams p) {
    constexpr int kVec = VecTraits<T>::kVec, kRows = kRowsAtOnce;
    grid_launch_dependents();
    const int lane = threadIdx.x & 7;
    const unsigned rows = (unsigned)p.B * p.Q * p.K * p.share;
    if constexpr (kScaled<T>) {
        const unsigned blocks = (rows + kDeltaRows - 1) / kDeltaRows;
        if (blockIdx.x >= blocks) return p.D <= 32 ? state_norms<T, 4>(p, blockIdx.x - blocks) : state_norms<T, 8>(p, blockIdx.x - blocks);
    }
    const unsigned first = blockIdx.x * kDeltaRows + (threadIdx.x >> 3);
    float sum[kRows] = {}, square[kRows] = {};
    for (int c = lane * kVec; c < p.D; c += 8 * kVec) {
        uint4 x[kRows], y[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const unsigned row = first + k * (kThreads / 8);
            const int64_t at = (int64_t)row * p.D + c;
            x[k] = row < rows ? ldg16(static_cast<const T *>(p.out) + at) : make_uint4(0, 0, 0, 0);
            y[k] = row < rows ? ldg16(static_cast<const T *>(p.grad_out) + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            float2 u[kVec / 2], v[kVec / 2];
            VecTraits<T>::unpack(x[k], u);
            VecTraits<T>::unpack(y[k], v);
#pragma unroll
            for (int i = 0; i < kVec / 2; ++i) {
                sum[k] += u[i].x * v[i].x + u[i].y * v[i].y;
                if constexpr (kScaled<T>) square[k] += v[i].x * v[i].x + v[i].y * v[i].y;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
            if constexpr (kScaled<T>) square[k] += __shfl_xor_sync(0xffffffffu, square[k], o);
        }
        const unsigned row = first + k * (kThreads / 8), token = row / (p.K * p.share), head = row - token * p.K * p.share;
        const unsigned b = token / p.Q, h = head / p.share;
        const int64_t at = ((int64_t)b * p.K + h) * p.R + (int64_t)(token - b * p.Q) * p.share + (head - h * p.share);
        if (lane == 0 && row < rows) {
            p.delta[at] = sum[k];
            if constexpr (kScaled<T>) p.row_norms[at] = p.lse[at] == INFINITY ? 0.f : sqrtf(square[k]);
        }
    }
}

// The largest norms and |delta| of a (sample, key head), by one CTA to 16 384 rows or states and eight at most, whose results the
// next kernel joins (262 144 rows of one head by one CTA: 30 us); what is not finite does not count.
__global__ void __launch_bounds__(1024) attention_bounds_kernel(const __grid_constant__ AttentionParams p) {
    __shared__ uint32_t warps[3][32];
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t bh = blockIdx.x / p.bound_ctas;
    const int first = (int)(blockIdx.x - bh * p.bound_ctas) * 1024 + threadIdx.x, step = 1024 * p.bound_ctas;
    const auto finite = [](float x) {
        const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
        return bits < 0x7f800000u ? bits : 0u;
    };
    uint32_t most[3] = {0, 0, 0};
#pragma unroll 4
    for (int i = first; i < p.R; i += step) {
        most[0] = max(most[0], finite(p.row_norms[bh * p.R + i]));
        most[1] = max(most[1], finite(p.delta[bh * p.R + i]));
    }
#pragma unroll 8
    for (int i = first; i < p.S; i += step) most[2] = max(most[2], finite(p.state_norms[bh * p.S + i]));
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        most[k] = __reduce_max_sync(0xffffffffu, most[k]);
        if ((threadIdx.x & 31) == 0) warps[k][threadIdx.x >> 5] = most[k];
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) most[k] = __reduce_max_sync(0xffffffffu, warps[k][threadIdx.x]);
    if (threadIdx.x == 0)
        (p.bound_ctas > 1 ? p.bound_parts : p.bounds)[blockIdx.x] =
            make_float4(__uint_as_float(most[0]), __uint_as_float(most[1]), __uint_as_float(most[2]), 0.f);
}

// a thread to a (sample, key head)
__global__ void __launch_bounds__(32) attention_bounds_join_kernel(const __grid_constant__ AttentionParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t bh = (int64_t)blockIdx.x * 32 + threadIdx.x;
    if (bh >= (int64_t)p.B * p.K) return;
    float4 most = p.bound_parts[bh * p.bound_ctas];
    for (int i = 1; i < p.bound_ctas; ++i) {
        const float4 x = p.bound_parts[bh * p.bound_ctas + i];
        most.x = fmaxf(most.x, x.x), most.y = fmaxf(most.y, x.y), most.z = fmaxf(most.z, x.z);
    }
    p.bounds[bh] = most;
}

// o = sum of 2^(L_i - L) o_i, a thread to four channels of a row
template <typename T>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const __grid_constant__ AttentionParams p) {
    grid_dependency_wait();
    const int lanes = p.D / 4;
    const int64_t rows = (int64_t)p.B * p.K * p.R;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / lanes;
    const int c = (int)(i - row * lanes) * 4;
    if (row >= rows) return;
    float top = -INFINITY;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_lse[s * rows + row]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = fast_exp2(p.part_lse[s * rows + row] - base);
        const float4 x = *reinterpret_cast<const float4 *>(p.part + (s * rows + row) * p.D + c);
        sum += w;
        o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t bh = row / p.R;
    const int r = (int)(row - bh * p.R), query = r / p.share, b = (int)(bh / p.K), h = (int)(bh - (int64_t)b * p.K);
    T *to = static_cast<T *>(p.out) +
            (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (r - query * p.share)) * p.D + c;
    to[0] = VecTraits<T>::from_float(o.x * inverse);
    to[1] = VecTraits<T>::from_float(o.y * inverse);
    to[2] = VecTraits<T>::from_float(o.z * inverse);
    to[3] = VecTraits<T>::from_float(o.w * inverse);
    if (c == 0) p.lse[row] = sum == 0.f ? INFINITY : base + log2f(sum);
}

// The same with a CTA to a row, its threads over the parts too: for many parts of few rows, where one thread's way
// through them is the time (78 parts of 8 rows: 8.9 us against 3).
constexpr int kManyParts = 16;
template <typename T>
__global__ void __launch_bounds__(128) attention_join_many_kernel(const __grid_constant__ AttentionParams p) {
    __shared__ float tops[4], weights[128];
    __shared__ float4 sums[128];
    grid_dependency_wait();
    const int64_t rows = (int64_t)p.B * p.K * p.R, row = blockIdx.x;
    const int lanes = p.D / 4, groups = 128 / lanes, group = threadIdx.x / lanes, c = (threadIdx.x - group * lanes) * 4;
    float top = -INFINITY;
    for (int s = threadIdx.x; s < p.splits; s += 128) top = fmaxf(top, p.part_lse[s * rows + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (group < groups)
        for (int s = group; s < p.splits; s += groups) {
            const float w = fast_exp2(p.part_lse[s * rows + row] - base);
            const float4 x = *reinterpret_cast<const float4 *>(p.part + (s * rows + row) * p.D + c);
            sum += w;
            o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
        }
    sums[threadIdx.x] = o, weights[threadIdx.x] = sum;
    __syncthreads();
    if (group != 0) return;
    for (int k = 1; k < groups; ++k) {
        const float4 x = sums[k * lanes + threadIdx.x];
        sum += weights[k * lanes + threadIdx.x];
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t bh = row / p.R;
    const int r = (int)(row - bh * p.R), query = r / p.share, b = (int)(bh / p.K), h = (int)(bh - (int64_t)b * p.K);
    T *to = static_cast<T *>(p.out) +
            (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (r - query * p.share)) * p.D + c;
    to[0] = VecTraits<T>::from_float(o.x * inverse);
    to[1] = VecTraits<T>::from_float(o.y * inverse);
    to[2] = VecTraits<T>::from_float(o.z * inverse);
    to[3] = VecTraits<T>::from_float(o.w * inverse);
    if (c == 0) p.lse[row] = sum == 0.f ? INFINITY : base + log2f(sum);
}

// gradients: the parts' sum, in the order of the parts; blockIdx.y: dk (or dq), dv
template <typename T, bool KEYS>
__global__ void __launch_bounds__(kThreads) attention_sum_kernel(const __grid_constant__ AttentionParams p) {
    grid_launch_dependents();
    grid_dependency_wait();
    const float *part = blockIdx.y == 0 ? p.part : p.part2;
    T *out = static_cast<T *>(!KEYS ? p.dq : blockIdx.y == 0 ? p.dk : p.dv);
    const int lanes = p.D / 4, X = KEYS ? p.S : p.R;
    const int64_t rows = (int64_t)p.B * p.K * X;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / lanes;
    const int c = (int)(i - row * lanes) * 4;
    if (row >= rows) return;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float4 x = *reinterpret_cast<const float4 *>(part + (s * rows + row) * p.D + c);
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    const int64_t bh = row / X;
    const int x = (int)(row - bh * X), b = (int)(bh / p.K), h = (int)(bh - (int64_t)b * p.K), query = x / p.share;
    T *to = out + (KEYS ? (((int64_t)b * p.S + x) * p.K + h) * p.D
                        : (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (x - query * p.share)) * p.D) + c;
    to[0] = VecTraits<T>::from_float(sum.x);
    to[1] = VecTraits<T>::from_float(sum.y);
    to[2] = VecTraits<T>::from_float(sum.z);
    to[3] = VecTraits<T>::from_float(sum.w);
}

unsigned blocks_for(int64_t threads) {
    return (unsigned)((threads + kThreads - 1) / kThreads);
}

template <typename T>
cudaError_t sum_typed(const AttentionParams &p, bool keys, cudaStream_t stream) {
    const dim3 grid(blocks_for((int64_t)p.B * p.K * (keys ? p.S : p.R) * (p.D / 4)), keys ? 2 : 1);
    return launch_dependent(keys ? attention_sum_kernel<T, true> : attention_sum_kernel<T, false>, grid, kThreads, 0, stream, p);
}

template <typename T>
cudaError_t join_typed(const AttentionParams &p, cudaStream_t stream) {
    const int64_t rows = (int64_t)p.B * p.K * p.R;
    if (p.splits >= kManyParts && rows < 148 * 64)
        return launch_dependent(attention_join_many_kernel<T>, dim3((unsigned)rows), 128, 0, stream, p);
    return launch_dependent(attention_join_kernel<T>, dim3(blocks_for(rows * (p.D / 4))), kThreads, 0, stream, p);
}

template <typename T>
cudaError_t delta_typed(const AttentionParams &p, cudaStream_t stream) {
    int64_t blocks = ((int64_t)p.B * p.K * p.R + kDeltaRows - 1) / kDeltaRows;
    const int64_t each = p.D <= 32 ? kStateRows<4> : kStateRows<8>;
    if constexpr (kScaled<T>) blocks += p.B * (((int64_t)p.S * p.K + each - 1) / each);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    attention_delta_kernel<T><<<(unsigned)blocks, kThreads, 0, stream>>>(p);
    cudaError_t e = cudaGetLastError();
    if constexpr (kScaled<T>) {
        if (e == cudaSuccess)
            e = launch_dependent(attention_bounds_kernel, dim3((unsigned)(p.B * p.K * p.bound_ctas)), 1024, 0, stream, p);
        if (e == cudaSuccess && p.bound_ctas > 1)
            e = launch_dependent(attention_bounds_join_kernel, dim3((unsigned)((p.B * p.K + 31) / 32)), 32, 0, stream, p);
    }
    return e;
}

}  // namespace

cudaError_t launch_attention_mask(const MaskParams &p, cudaStream_t stream) {
    if (p.mask == nullptr) {
        attention_padding_kernel<<<(unsigned)p.B, 1024, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const int64_t tasks = (int64_t)p.B * p.H * p.Q * ((p.W + 31) / 32);
    const int64_t grid = std::min<int64_t>((tasks + kThreads / 32 - 1) / (kThreads / 32), 148 * 64);
    attention_mask_kernel<<<(unsigned)grid, kThreads, 0, stream>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess)
        e = launch_dependent(attention_mask_any_kernel, dim3((unsigned)(p.B * p.KW * ((p.W + 31) / 32))), 1024, 0, stream, p);
    if (e == cudaSuccess) e = launch_dependent(attention_list_kernel, dim3((unsigned)(p.B * p.KW)), 1024, 0, stream, p);
    return e;
}

cudaError_t launch_attention_terms(const TermsParams &p, cudaStream_t stream) {
    int64_t most = 0;
    for (int i = 0; i < p.tensors; ++i) most = std::max(most, (int64_t)p.B * p.of[i].tokens * p.of[i].heads * ((p.D + 7) / 8));
    const int64_t grid = std::min<int64_t>((most + kThreads - 1) / kThreads, 148 * 32);
    return launch_dependent(attention_terms_kernel, dim3((unsigned)grid, p.tensors), kThreads, 0, stream, p);
}

cudaError_t launch_attention_delta(const AttentionParams &p, int dtype, cudaStream_t stream) {
    return dtype == 0 ? delta_typed<float>(p, stream)
           : dtype == 1 ? delta_typed<__half>(p, stream) : delta_typed<__nv_bfloat16>(p, stream);
}
cudaError_t launch_attention_join(const AttentionParams &p, int dtype, cudaStream_t stream) {
    return dtype == 0 ? join_typed<float>(p, stream)
           : dtype == 1 ? join_typed<__half>(p, stream) : join_typed<__nv_bfloat16>(p, stream);
}
cudaError_t launch_attention_sum(const AttentionParams &p, bool keys, int dtype, cudaStream_t stream) {
    return dtype == 0 ? sum_typed<float>(p, keys, stream)
           : dtype == 1 ? sum_typed<__half>(p, keys, stream) : sum_typed<__nv_bfloat16>(p, keys, stream);
}

}  // namespace msda_b200
