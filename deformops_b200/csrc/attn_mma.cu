// Cross attention backward with warp-level matrix instructions, for more than 64 query heads to a key head: whole tokens
// of so many rows fill no tile of the kernel of attn_tc_backward.cu.  2 x 64 queries of 130 heads over 4096 states
// of one head of 64: float32 1.7 ms (0.16 of products at what the GPU sustains), bf16 0.76.
//
// One kernel template in two forms.  "keys" holds 64 states and walks the rows (dk, dv), the other holds 64 rows and
// walks the states (dq); the weights are formed again in both, so that every gradient is summed by one warp in a
// fixed order: no atomics, the same bits on every run.
//
// float32 operands go through the tensor cores as two terms of tf32 (x = hi + lo, 11 bits each);
// lo * hi + hi * lo + hi * hi leaves 2^-21 of a product, sums are float32.  16-bit operands take
// m16n8k16; the weights, and ds, are rounded to the type there (half a step each, the step of the
// result's own rounding) and everything else stays float32.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "warp_mma.cuh"

namespace msda_b200 {

namespace {

constexpr int kThreads = 128;      // four warps

__device__ __forceinline__ uint32_t smem_address(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void cp_async16(void *to, const void *from, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_address(to)), "l"(from),
                 "r"(valid ? 16 : 0));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// rows of a tile in shared memory are DP elements and 16 bytes apart, so that eight rows (ldmatrix),
// and 8 x 4 or 4 x 8 single floats, fall on distinct banks
template <typename T, int DP>
constexpr int kPitch = DP + 16 / sizeof(T);

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_address(p)));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_address(p)));
}

// acc (16 x 8N) = A B^T: A the warp's 16 rows, B 8N rows, DP columns each
template <typename T, int DP, int N>
__device__ __forceinline__ void product_nt(float (&acc)[N][4], const T *a, const T *b) {
    constexpr int P = kPitch<T, DP>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    if constexpr (sizeof(T) == 2) {
        const T *pa = a + (lane & 15) * P + (lane >> 4) * 8;
        const T *pb = b + ((lane >> 4) * 8 + (lane & 7)) * P + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int k = 0; k < DP; k += 16) {
            uint32_t fa[4];
            ldmatrix4(fa, pa + k);
#pragma unroll
            for (int n = 0; n < N; n += 2) {
                uint32_t fb[4];
                ldmatrix4(fb, pb + n * 8 * P + k);
                mma16<T>(acc[n], fa, fb[0], fb[1]);
                mma16<T>(acc[n + 1], fa, fb[2], fb[3]);
            }
        }
    } else {
#pragma unroll 4
        for (int k = 0; k < DP; k += 8) {
            uint32_t ah[4], al[4];
            split_tf32(a[g * P + k + t], ah[0], al[0]);
            split_tf32(a[(g + 8) * P + k + t], ah[1], al[1]);
            split_tf32(a[g * P + k + t + 4], ah[2], al[2]);
            split_tf32(a[(g + 8) * P + k + t + 4], ah[3], al[3]);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                uint32_t bh[2], bl[2];
                split_tf32(b[(n * 8 + g) * P + k + t], bh[0], bl[0]);
                split_tf32(b[(n * 8 + g) * P + k + t + 4], bh[1], bl[1]);
                mma_tf32x3(acc[n], ah, al, bh, bl);
            }
        }
    }
}

// acc (16 x DP) += W B: W 16 x 8N in accumulator layout, B 8N rows of DP columns
template <typename T, int DP, int N>
__device__ __forceinline__ void add_product_nn(float (&acc)[DP / 8][4], const float (&w)[N][4], const T *b) {
    constexpr int P = kPitch<T, DP>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (sizeof(T) == 2) {
        const T *pb = b + (lane & 15) * P + (lane >> 4) * 8;
#pragma unroll
        for (int n = 0; n < N; n += 2) {
            const uint32_t fa[4] = {VecTraits<T>::pack2(make_float2(w[n][0], w[n][1])),
                                    VecTraits<T>::pack2(make_float2(w[n][2], w[n][3])),
                                    VecTraits<T>::pack2(make_float2(w[n + 1][0], w[n + 1][1])),
                                    VecTraits<T>::pack2(make_float2(w[n + 1][2], w[n + 1][3]))};
#pragma unroll
            for (int d = 0; d < DP / 8; d += 2) {
                uint32_t fb[4];
                ldmatrix4_trans(fb, pb + n * 8 * P + d * 8);
                mma16<T>(acc[d], fa, fb[0], fb[1]);
                mma16<T>(acc[d + 1], fa, fb[2], fb[3]);
            }
        }
    } else {
        // the product's k runs over rows in any order: position t is row 2t, position t + 4 row 2t + 1,
        // which is where the accumulator layout has them
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t ah[4], al[4];
            split_tf32(w[n][0], ah[0], al[0]);
            split_tf32(w[n][2], ah[1], al[1]);
            split_tf32(w[n][1], ah[2], al[2]);
            split_tf32(w[n][3], ah[3], al[3]);
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
                uint32_t bh[2], bl[2];
                split_tf32(b[(n * 8 + 2 * t) * P + d * 8 + g], bh[0], bl[0]);
                split_tf32(b[(n * 8 + 2 * t + 1) * P + d * 8 + g], bh[1], bl[1]);
                mma_tf32x3(acc[d], ah, al, bh, bl);
            }
        }
    }
}

// The same with sums kept apart for float32: a matrix instruction cuts its sum off where it should round,
// always towards zero, which over the thousands of instructions of a long axis adds up (17 821 states: 1.6e-5 of
// the result, against 1e-6 so).  A tile's product starts from zero and is added with rounding.
template <typename T, int DP, int N>
__device__ __forceinline__ void product_nn(float (&acc)[DP / 8][4], const float (&w)[N][4], const T *b) {
    if constexpr (sizeof(T) == 4) {
        float tile[DP / 8][4];
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) tile[d][0] = tile[d][1] = tile[d][2] = tile[d][3] = 0.f;
        add_product_nn<T, DP, N>(tile, w, b);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[d][e] += tile[d][e];
    } else {
        add_product_nn<T, DP, N>(acc, w, b);
    }
}

// rows first .. first + ROWS of k or v to shared memory; rows that nobody may see become zeros
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_states(T *to, const T *base, int64_t stride, int first, int S, int D,
                                            const uint32_t *words) {
    constexpr int kVec = 16 / sizeof(T), kChunks = DP / kVec;
    for (int i = threadIdx.x; i < ROWS * kChunks; i += kThreads) {
        const int row = i / kChunks, chunk = i - row * kChunks, state = first + row;
        const bool valid = chunk * kVec < D && ((key_word(words, S, state >> 5) >> (state & 31)) & 1);
        cp_async16(to + row * kPitch<T, DP> + chunk * kVec, valid ? base + state * stride + chunk * kVec : base, valid);
    }
}

// packed rows first .. first + ROWS of a (B, Q, G, D) tensor
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_rows(T *to, const T *base, const int64_t (&strides)[3], const AttentionParams &p,
                                          int b, int h, int first) {
    constexpr int kVec = 16 / sizeof(T), kChunks = DP / kVec;
    for (int i = threadIdx.x; i < ROWS * kChunks; i += kThreads) {
        const int row = i / kChunks, chunk = i - row * kChunks, r = first + row;
        const bool valid = chunk * kVec < p.D && r < p.R;
        cp_async16(to + row * kPitch<T, DP> + chunk * kVec,
                   valid ? base + row_offset(strides, p.share, b, h, r) + chunk * kVec : base, valid);
    }
}

// the first tile of `tiles` (each WORDS mask words) from t on in which some state may be seen
template <int WORDS>
__device__ __forceinline__ int next_tile(const uint32_t *words, int S, int t, int end) {
    if (words == nullptr) return t;
    for (; t < end; ++t) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) any |= 32 * (t * WORDS + i) < S ? __ldg(words + t * WORDS + i) : 0;
        if (any) return t;
    }
    return end;
}

// KEYS: holds 64 states, walks the rows, sums dv = p^T do and dk = ds^T q.  Otherwise holds 64 rows,
// walks the states and sums dq = ds k.
template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads) attention_backward_mma_kernel(const __grid_constant__ AttentionParams p) {
    constexpr int BX = 64, BN = DP == 128 ? 32 : 64, N = BN / 8, P = kPitch<T, DP>;
    extern __shared__ __align__(16) unsigned char smem[];
    T *const x0 = reinterpret_cast<T *>(smem);         // k or q
    T *const x1 = x0 + BX * P;                         // v or do
    T *const y0 = x1 + BX * P;                         // two stages: q or k
    T *const y1 = y0 + 2 * BN * P;                     // do or v
    float *const s_lse = reinterpret_cast<float *>(y1 + 2 * BN * P);      // two stages of BN, KEYS only
    float *const s_delta = s_lse + 2 * BN;
    uint32_t *const s_words = reinterpret_cast<uint32_t *>(s_delta + 2 * BN);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

    grid_launch_dependents();
    grid_dependency_wait();
    const int x_tiles = ((KEYS ? p.S : p.R) + BX - 1) / BX;
    int64_t i = blockIdx.x;
    const int first = (int)(i % x_tiles) * BX;
    i /= x_tiles;
    const int part = (int)(i % p.splits);
    const int64_t bh = i / p.splits;
    const int b = (int)(bh / p.K), h = (int)(bh % p.K);
    const T *k = static_cast<const T *>(p.k) + b * p.ks[0] + h * p.ks[2];
    const T *v = static_cast<const T *>(p.v) + b * p.vs[0] + h * p.vs[2];
    const int64_t gs[3] = {(int64_t)p.Q * p.K * p.share * p.D, (int64_t)p.K * p.share * p.D, p.D};
    const uint32_t *words = key_words_of(p, b, h);
    const int all_tiles = ((KEYS ? p.R : p.S) + BN - 1) / BN;
    int end = min(all_tiles, (part + 1) * p.tiles);
    if (KEYS && next_tile<BX / 32>(words, p.S, first / BX, first / BX + 1) != first / BX) end = 0;   // nobody sees them

    auto skip = [&](int tile) { return KEYS ? tile : next_tile<BN / 32>(words, p.S, tile, end); };
    auto load = [&](int tile, int stage) {
        if constexpr (KEYS) {
            load_rows<T, DP, BN>(y0 + stage * BN * P, static_cast<const T *>(p.q), p.qs, p, b, h, tile * BN);
            load_rows<T, DP, BN>(y1 + stage * BN * P, static_cast<const T *>(p.grad_out), gs, p, b, h, tile * BN);
            for (int c = threadIdx.x; c < BN; c += kThreads) {
                const int r = tile * BN + c;
                s_lse[stage * BN + c] = r < p.R ? p.lse[bh * p.R + r] - (kScaled<T> ? kWeightExponent : 0.f) : INFINITY;
                s_delta[stage * BN + c] = r < p.R ? p.delta[bh * p.R + r] : 0.f;
                if (p.row_words != nullptr)
#pragma unroll
                    for (int w = 0; w < BX / 32; ++w)
                        s_words[(stage * BN + c) * (BX / 32) + w] =
                            r < p.R ? __ldg(row_words_of(p, b, h, r) + first / 32 + w) : 0;
            }
        } else {
            load_states<T, DP, BN>(y0 + stage * BN * P, k, p.ks[1], tile * BN, p.S, p.D, words);
            load_states<T, DP, BN>(y1 + stage * BN * P, v, p.vs[1], tile * BN, p.S, p.D, words);
        }
    };

    int tile = skip(part * p.tiles);
    if constexpr (KEYS) {
        load_states<T, DP, BX>(x0, k, p.ks[1], first, p.S, p.D, words);
        load_states<T, DP, BX>(x1, v, p.vs[1], first, p.S, p.D, words);
    } else {
        load_rows<T, DP, BX>(x0, static_cast<const T *>(p.q), p.qs, p, b, h, first);
        load_rows<T, DP, BX>(x1, static_cast<const T *>(p.grad_out), gs, p, b, h, first);
    }
    if (tile < end) load(tile, 0);
    cp_async_commit();

    const int x_row = first + warp * 16 + g;           // and x_row + 8
    float lse[2] = {INFINITY, INFINITY}, delta[2] = {0.f, 0.f};
    float grow[2] = {1.f, 1.f}, unscale[2] = {p.scale, p.scale};     // of dS, and back (float16)
    const uint32_t *rw[2] = {nullptr, nullptr};
    bool seen[2] = {false, false};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = x_row + 8 * half;
        if constexpr (KEYS) {
            seen[half] = (key_word(words, p.S, r >> 5) >> (r & 31)) & 1;
        } else if (r < p.R) {
            lse[half] = p.lse[bh * p.R + r];
            delta[half] = p.delta[bh * p.R + r];
            rw[half] = row_words_of(p, b, h, r);
        }
        if (kScaled<T> && r < (KEYS ? p.S : p.R)) {
            const float by = KEYS ? state_scale(p, bh, r) : row_scale(p, bh, r);
            grow[half] = KEYS ? by * (1.f / kWeightScale) : by, unscale[half] = p.scale / by;
        }
    }

    float a0[KEYS ? DP / 8 : 1][4], a1[DP / 8][4];
#pragma unroll
    for (int d = 0; d < DP / 8; ++d) {
        if constexpr (KEYS) a0[d][0] = a0[d][1] = a0[d][2] = a0[d][3] = 0.f;
        a1[d][0] = a1[d][1] = a1[d][2] = a1[d][3] = 0.f;
    }

    for (int stage = 0; tile < end; stage ^= 1) {
        const int next = skip(tile + 1);
        if (next < end) load(next, stage ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();

        float s[N][4], ds[N][4];
        product_nt<T, DP, N>(s, x0 + warp * 16 * P, y0 + stage * BN * P);
        product_nt<T, DP, N>(ds, x1 + warp * 16 * P, y1 + stage * BN * P);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int col = n * 8 + 2 * t + e, j = 2 * half + e;
                    bool may;
                    float row_lse, row_delta;
                    if constexpr (KEYS) {
                        const int c = stage * BN + col, key = warp * 16 + g + 8 * half;
                        may = p.row_words != nullptr ? (s_words[c * (BX / 32) + (key >> 5)] >> (key & 31)) & 1 : seen[half];
                        row_lse = s_lse[c], row_delta = s_delta[c];
                    } else {
                        const int state = tile * BN + col;
                        may = ((rw[half] != nullptr ? __ldg(rw[half] + (state >> 5)) : key_word(words, p.S, state >> 5)) >>
                               (state & 31)) & 1;
                        row_lse = lse[half], row_delta = delta[half];
                    }
                    s[n][j] = may ? fast_exp2(s[n][j] * p.scale_log2 - row_lse) : 0.f;
                    ds[n][j] = may ? s[n][j] * ((ds[n][j] - row_delta) * grow[half]) : 0.f;
                }
        if constexpr (KEYS) product_nn<T, DP, N>(a0, s, y1 + stage * BN * P);
        product_nn<T, DP, N>(a1, ds, y0 + stage * BN * P);
        __syncthreads();
        tile = next;
    }
    cp_async_wait<0>();

#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int x = x_row + 8 * half;
        if (x >= (KEYS ? p.S : p.R)) continue;
        const int64_t rows = (int64_t)p.B * p.K * (KEYS ? p.S : p.R);
        const int64_t at = bh * (KEYS ? p.S : p.R) + x;
        const int query = x / p.share;
        const int64_t final_at = KEYS ? (((int64_t)b * p.S + x) * p.K + h) * p.D
                                      : (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (x - query * p.share)) * p.D;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
            const int c = d * 8 + 2 * t;
            if (c >= p.D) continue;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float grad = a1[d][2 * half + e] * unscale[half];
                float grad_value = 0.f;
                if constexpr (KEYS) grad_value = a0[d][2 * half + e] * (kScaled<T> ? 1.f / kWeightScale : 1.f);
                if (p.splits > 1) {
                    p.part[(part * rows + at) * p.D + c + e] = grad;
                    if constexpr (KEYS) p.part2[(part * rows + at) * p.D + c + e] = grad_value;
                } else {
                    static_cast<T *>(KEYS ? p.dk : p.dq)[final_at + c + e] = VecTraits<T>::from_float(grad);
                    if constexpr (KEYS) static_cast<T *>(p.dv)[final_at + c + e] = VecTraits<T>::from_float(grad_value);
                }
            }
        }
    }
}

// more than 48 KB have to be asked for: with every call, captured ones too, since devices do not share it
template <typename Kernel>
cudaError_t launch(Kernel kernel, int64_t grid, size_t smem, cudaStream_t stream, const AttentionParams &p) {
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(kernel, dim3((unsigned)grid), kThreads, smem, stream, p);
}

template <typename T, int DP, bool KEYS>
cudaError_t backward(const AttentionParams &p, cudaStream_t stream) {
    constexpr int BN = DP == 128 ? 32 : 64;
    constexpr size_t smem = (size_t)(128 + 4 * BN) * kPitch<T, DP> * sizeof(T) + 4 * BN * sizeof(float) +
                            (size_t)2 * BN * 2 * sizeof(uint32_t);
    const int64_t grid = (int64_t)p.B * p.K * p.splits * (((KEYS ? p.S : p.R) + 63) / 64);
    return launch(attention_backward_mma_kernel<T, DP, KEYS>, grid, smem, stream, p);
}

template <typename T, int DP>
cudaError_t backward_side(const AttentionParams &p, bool keys, cudaStream_t stream) {
    return keys ? backward<T, DP, true>(p, stream) : backward<T, DP, false>(p, stream);
}

template <typename T>
cudaError_t backward_typed(const AttentionParams &p, bool keys, cudaStream_t stream) {
    return p.D <= 32 ? backward_side<T, 32>(p, keys, stream)
           : p.D <= 64 ? backward_side<T, 64>(p, keys, stream) : backward_side<T, 128>(p, keys, stream);
}

}  // namespace

cudaError_t launch_attention_backward_mma(const AttentionParams &p, int dtype, bool keys, cudaStream_t stream) {
    return dtype == 0 ? backward_typed<float>(p, keys, stream)
           : dtype == 1 ? backward_typed<__half>(p, keys, stream) : backward_typed<__nv_bfloat16>(p, keys, stream);
}

}  // namespace msda_b200
