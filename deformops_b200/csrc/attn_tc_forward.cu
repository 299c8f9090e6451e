// Cross attention forward on the fifth-generation tensor cores, 16-bit types.
//
// A CTA holds NQ tiles of 128 rows and walks the states 128 at a time.  One thread has TMA bring the
// tiles of k and v, one thread issues the products, and four warps per row tile do the softmax, a
// thread to a row: scores come from tensor memory, weights go back there as the left operand of the
// second product, whose sums stay in tensor memory until the end.
//
//   S = q k^T (tensor memory, 128 columns)   P = exp2(c S - m) (64 columns, 16-bit)   O += P v
//
// The running maximum is only raised when a row would leave exp2's range of 2^8 above it: then the
// row's sums in tensor memory are scaled, which is rare after the first tiles, and exact in between (a
// weight of up to 2^8 rounds like one of 1).
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace msda_b200 {

namespace {

constexpr int kTileRows = 128, kTileStates = 128;

template <int DP>
constexpr int kStages = DP == 32 ? 4 : 2;

template <int DP, int NQ>
struct Shared {
    alignas(1024) unsigned char q[NQ][kTileRows * DP * 2];
    alignas(1024) unsigned char k[kStages<DP>][kTileStates * DP * 2];
    alignas(1024) unsigned char v[kStages<DP>][kTileStates * DP * 2];
    uint64_t k_full[kStages<DP>], k_free[kStages<DP>], v_full[kStages<DP>], v_free[kStages<DP>];
    uint64_t s_full[NQ], s_free[NQ], p_full[NQ], o_full[NQ];
    uint32_t tmem;
};

__device__ __forceinline__ uint4 tile_words(const uint32_t *words, int S, int tile) {
    if (words != nullptr) return __ldg(reinterpret_cast<const uint4 *>(words) + tile);
    return make_uint4(key_word(nullptr, S, 4 * tile), key_word(nullptr, S, 4 * tile + 1), key_word(nullptr, S, 4 * tile + 2),
                      key_word(nullptr, S, 4 * tile + 3));
}

// the first tile from t on in which some state may be seen
__device__ __forceinline__ int next_tile(const uint32_t *words, int t, int end) {
    if (words == nullptr) return t;
    for (; t < end; ++t) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(words) + t);
        if (w.x | w.y | w.z | w.w) return t;
    }
    return end;
}

template <typename T, int DP, int NQ>
__global__ void __launch_bounds__(NQ * 128 + 128, NQ == 1 ? 2 : 1)
    attention_forward_tc_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ tc::TensorMap km,
                                const __grid_constant__ tc::TensorMap vm) {
    using namespace tc;
    // columns of tensor memory of one row tile: S, P, O.  At 128 channels P takes the place of S, and the next
    // scores wait for the product that reads it.
    constexpr bool kAlias = DP == 128;
    constexpr uint32_t kS = 0, kP = kAlias ? 0 : 128, kO = kAlias ? 128 : 192, kColumns = 256;
    constexpr int ST = kStages<DP>;
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    extern __shared__ __align__(1024) unsigned char raw[];
    auto &sm = *reinterpret_cast<Shared<DP, NQ> *>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int row_tiles = (p.R + NQ * kTileRows - 1) / (NQ * kTileRows);
    int64_t i = blockIdx.x;
    const int first = (int)(i % row_tiles) * NQ * kTileRows;
    i /= row_tiles;
    const int part = (int)(i % p.splits);
    const int64_t bh = i / p.splits;
    const int b = (int)(bh / p.K), h = (int)(bh % p.K);
    const uint32_t *words = key_words_of(p, b, h);
    const int end = min((p.S + kTileStates - 1) / kTileStates, (part + 1) * p.tiles);

    if (warp == 4 * NQ) tmem_alloc(&sm.tmem, NQ * kColumns);
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            barrier_init(&sm.k_full[s], 1), barrier_init(&sm.k_free[s], 1);
            barrier_init(&sm.v_full[s], 1), barrier_init(&sm.v_free[s], 1);
        }
        for (int q = 0; q < NQ; ++q) {
            barrier_init(&sm.s_full[q], 1), barrier_init(&sm.s_free[q], 128);
            barrier_init(&sm.p_full[q], 128), barrier_init(&sm.o_full[q], 1);
        }
    }
    if (warp < 4 * NQ) {
        // a thread to a row of q
        const int r = first + threadIdx.x;
        const T *q = static_cast<const T *>(p.q) + (r < p.R ? row_offset(p.qs, p.share, b, h, r) : 0);
        unsigned char *to = sm.q[warp >> 2];
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
            const uint4 x = r < p.R && c * 8 < p.D ? ldg16(q + c * 8) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(to + swizzled<DP, kTileRows>(threadIdx.x & 127, c)) = x;
        }
        fence_async_shared();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm.tmem;
    bool fine = true;

    if (warp < 4 * NQ) {
        registers_up<NQ == 1 ? 200 : 224>();
        const int q = warp >> 2;
        const uint32_t mine = tmem + q * kColumns + ((uint32_t)(warp & 3) << 21);
        const int r = first + threadIdx.x;
        const bool idle = first + (warp << 5) >= p.R;              // a whole warp behind the last row
        const uint32_t *rw = r < p.R ? row_words_of(p, b, h, r) : nullptr;
        float m = -INFINITY, l = 0.f;
        int done = 0;
        for (int tile = next_tile(words, part * p.tiles, end); fine && tile < end; ++done) {
            const int next = next_tile(words, tile + 1, end);
            const uint4 see = rw != nullptr ? __ldg(reinterpret_cast<const uint4 *>(rw) + tile) : tile_words(words, p.S, tile);
            fine = barrier_wait(&sm.s_full[q], done & 1);
            if (!fine) break;
            fence_after();
            if (idle) {
                if constexpr (!kAlias) {
                    barrier_arrive(&sm.s_free[q]);
                    // (not before the other warps' weights of the tile before have been counted)
                    if (done > 0) fine = barrier_wait(&sm.o_full[q], (done - 1) & 1);
                }
                barrier_arrive(&sm.p_full[q]);
                tile = next;
                continue;
            }
            uint32_t s[4][32];
#pragma unroll
            for (int j = 0; j < 4; ++j) tmem_load32(s[j], mine + kS + 32 * j);
            tmem_wait_load();
#pragma unroll
            for (int j = 0; j < 4; ++j) loaded(s[j]);
            if constexpr (!kAlias) {
                fence_before();
                barrier_arrive(&sm.s_free[q]);
            }
            if (!__all_sync(0xffffffffu, (see.x & see.y & see.z & see.w) == 0xffffffffu)) {
                const uint32_t w[4] = {see.x, see.y, see.z, see.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(w[j] & (1u << c))) s[j][c] = 0xff800000u;        // -inf
            }
            float top[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                top[j] = __uint_as_float(s[j][0]);
#pragma unroll
                for (int c = 1; c < 32; ++c) top[j] = fmaxf(top[j], __uint_as_float(s[j][c]));
            }
            const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
            const bool raise = best > m + 8.f || (m == -INFINITY && best > m);
            bool waited = kAlias || done == 0;       // the product before has read P and added to O
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? best : m;
                const float keep = to == -INFINITY ? 1.f : fast_exp2(m - to);
                m = to;
                l *= keep;
                if (done > 0) {
                    if (!waited) {
                        fine = barrier_wait(&sm.o_full[q], (done - 1) & 1);
                        fence_after();
                        waited = true;
                    }
#pragma unroll
                    for (int d = 0; d < DP; d += 32) {
                        uint32_t o[32];
                        tmem_load32(o, mine + kO + d);
                        tmem_wait_load();
                        loaded(o);
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
                        tmem_store32(mine + kO + d, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m;
            const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
            float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
            const float2 one = make_float2(1.f, 1.f);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                uint32_t w[32];
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    float2 x = make_float2(-base, -base);
                    ffma2(x, make_float2(__uint_as_float(s[j + (c >> 5)][c & 31]), __uint_as_float(s[j + (c >> 5)][(c & 31) + 1])),
                          scale2);
                    x.x = fast_exp2(x.x), x.y = fast_exp2(x.y);
                    ffma2(sum[(c >> 1) & 1], x, one);
                    w[c >> 1] = VecTraits<T>::pack2(x);
                }
                if (!waited) {
                    fine = barrier_wait(&sm.o_full[q], (done - 1) & 1) && fine;
                    fence_after();
                    waited = true;
                }
                tmem_store32(mine + kP + 16 * j, w);
            }
            l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_wait_store();
            fence_before();
            barrier_arrive(&sm.p_full[q]);
            tile = next;
        }
        // results: the rows of O over their sums
        if (done > 0 && !idle) {
            fine = barrier_wait(&sm.o_full[q], (done - 1) & 1) && fine;
            fence_after();
        }
        const float inverse = !fine ? NAN : l > 0.f || l != l ? 1.f / l : 0.f;
        const float lse = l == 0.f ? (p.splits > 1 ? -INFINITY : INFINITY) : m + log2f(l);
        const int64_t at = bh * p.R + r, rows = (int64_t)p.B * p.K * p.R;
        const int query = r / p.share;
        T *out = static_cast<T *>(p.out) + (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (r - query * p.share)) * p.D;
        float *parts = p.part + (part * rows + at) * p.D;
        if (r < p.R) (p.splits > 1 ? p.part_lse + part * rows : p.lse)[at] = lse;
        if (!idle) {
#pragma unroll
            for (int d = 0; d < DP; d += 32) {
                uint32_t o[32];
                if (done > 0) {
                    tmem_load32(o, mine + kO + d);
                    tmem_wait_load();
                    loaded(o);
                }
                float2 x[16];
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    x[c] = done > 0 ? make_float2(__uint_as_float(o[2 * c]) * inverse, __uint_as_float(o[2 * c + 1]) * inverse)
                                    : make_float2(0.f, 0.f);
                if (r < p.R && p.splits > 1) {
#pragma unroll
                    for (int c = 0; c < 16; c += 2)
                        if (d + 2 * c < p.D)
                            *reinterpret_cast<float4 *>(parts + d + 2 * c) = make_float4(x[c].x, x[c].y, x[c + 1].x, x[c + 1].y);
                } else if (r < p.R) {
#pragma unroll
                    for (int c = 0; c < 16; c += 4)
                        if (d + 2 * c < p.D) {
                            const float2 y[4] = {x[c], x[c + 1], x[c + 2], x[c + 3]};
                            *reinterpret_cast<uint4 *>(out + d + 2 * c) = VecTraits<T>::pack(y);
                        }
                }
            }
        }
        fence_before();
    } else {
        registers_down<56>();
        if (warp == 4 * NQ && lane == 0) {
            int n = 0;
            for (int tile = next_tile(words, part * p.tiles, end); fine && tile < end; ++n) {
                const int stage = n % ST, turn = n / ST;
                if (turn > 0) fine = barrier_wait(&sm.k_free[stage], (turn - 1) & 1);
                if (fine) {
                    barrier_expect(&sm.k_full[stage], kTileStates * DP * 2);
                    load_rows<DP, kTileStates>(sm.k[stage], km, &sm.k_full[stage], b, h, tile * kTileStates);
                }
                if (fine && turn > 0) fine = barrier_wait(&sm.v_free[stage], (turn - 1) & 1);
                if (fine) {
                    barrier_expect(&sm.v_full[stage], kTileStates * DP * 2);
                    load_rows<DP, kTileStates>(sm.v[stage], vm, &sm.v_full[stage], b, h, tile * kTileStates);
                }
                tile = next_tile(words, tile + 1, end);
            }
            // nothing may still be on its way when the CTA ends
            for (int s = 0; s < ST; ++s) {
                const int turns = (n - s + ST - 1) / ST;
                if (turns > 0 && !fine) barrier_wait(&sm.k_full[s], (turns - 1) & 1), barrier_wait(&sm.v_full[s], (turns - 1) & 1);
            }
        } else if (warp == 4 * NQ + 1) {
            constexpr uint32_t kScores = instruction(kBf16, 128, 128, false, false);
            constexpr uint32_t kOut = instruction(kBf16, 128, DP, false, true);
            constexpr int kRow = kRowBytes<DP>;
            int before = -1, n = 0;
            // n-th tile: its scores, then the product with the weights of the tile before
            for (int tile = next_tile(words, part * p.tiles, end); fine && (tile < end || before >= 0); ++n) {
                const bool scores = tile < end, weights = before >= 0;
                const int stage = n % ST, last = (n + ST - 1) % ST;
                if (scores) fine = barrier_wait(&sm.k_full[stage], (n / ST) & 1);
                if (weights) {
                    fine = fine && barrier_wait(&sm.v_full[last], ((n - 1) / ST) & 1);
                    if (words != nullptr && fine) {
                        // rows of v that nobody may see: whatever they hold, their weight is 0 and has to stay it
                        const uint4 see = __ldg(reinterpret_cast<const uint4 *>(words) + before);
                        if ((see.x & see.y & see.z & see.w) != 0xffffffffu) {
                            const uint32_t w[4] = {see.x, see.y, see.z, see.w};
                            constexpr int kChunks = DP / 8;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                for (int c = lane; c < 32 * kChunks; c += 32)
                                    if (!((w[j] >> (c / kChunks)) & 1))
                                        *reinterpret_cast<uint4 *>(sm.v[last] + swizzled<DP, kTileStates>(32 * j + c / kChunks, c % kChunks)) =
                                            make_uint4(0, 0, 0, 0);
                            fence_async_shared();
                            __syncwarp();
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const uint32_t at = tmem + q * kColumns;
                    const auto issue_scores = [&] {
                        if (!kAlias && n > 0) fine = fine && barrier_wait(&sm.s_free[q], (n - 1) & 1);
                        fence_after();
                        if (fine && lane == 0) {
                            const uint32_t qa = smem_address(sm.q[q]), ka = smem_address(sm.k[stage]);
#pragma unroll
                            for (int d = 0; d < DP; d += 16) {
                                const uint32_t off = (d >> 6) * kTileRows * 128 + (d & 63) * 2;
                                mma(at + kS, descriptor<kRow>(qa + off, 16), descriptor<kRow>(ka + off, 16), kScores, d > 0);
                            }
                            commit(&sm.s_full[q]);
                            if (q == NQ - 1) commit(&sm.k_free[stage]);
                        }
                    };
                    const auto issue_weights = [&] {
                        fine = fine && barrier_wait(&sm.p_full[q], (n - 1) & 1);
                        fence_after();
                        if (fine && lane == 0) {
                            const uint32_t va = smem_address(sm.v[last]);
#pragma unroll
                            for (int j = 0; j < kTileStates; j += 16)
                                mma_ts(at + kO, at + kP + j / 2, descriptor<kRow>(va + j * kRow, kTileStates * 128), kOut,
                                       n > 1 || j > 0);
                            commit(&sm.o_full[q]);
                            if (q == NQ - 1) commit(&sm.v_free[last]);
                        }
                    };
                    if constexpr (kAlias) {
                        if (weights) issue_weights();
                        if (scores) issue_scores();
                    } else {
                        if (scores) issue_scores();
                        if (weights) issue_weights();
                    }
                }
                before = scores ? tile : -1;
                if (scores) tile = next_tile(words, tile + 1, end);
            }
        }
    }
    __syncthreads();
    if (warp == 4 * NQ) {
        fence_after();
        tmem_free(tmem, NQ * kColumns);
    }
}

template <typename T, int DP, int NQ>
cudaError_t launch(const AttentionParams &p, cudaStream_t stream) {
    tc::TensorMap km, vm;
    if (!tc::make_map<T, DP>(km, p.k, p.ks, p.B, p.S, p.K, 1, p.D, kTileStates) ||
        !tc::make_map<T, DP>(vm, p.v, p.vs, p.B, p.S, p.K, 1, p.D, kTileStates))
        return cudaErrorNotSupported;
    const auto kernel = attention_forward_tc_kernel<T, DP, NQ>;
    constexpr size_t smem = sizeof(Shared<DP, NQ>);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)p.B * p.K * p.splits * ((p.R + NQ * kTileRows - 1) / (NQ * kTileRows));
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    kernel<<<(unsigned)grid, NQ * 128 + 128, smem, stream>>>(p, km, vm);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, int row_tiles, cudaStream_t stream) {
    if (p.D <= 32) return row_tiles == 1 ? launch<T, 32, 1>(p, stream) : launch<T, 32, 2>(p, stream);
    if (p.D <= 64) return row_tiles == 1 ? launch<T, 64, 1>(p, stream) : launch<T, 64, 2>(p, stream);
    return launch<T, 128, 2>(p, stream);
}

}  // namespace

cudaError_t launch_attention_forward_tc(const AttentionParams &p, int dtype, int row_tiles, cudaStream_t stream) {
    return dtype == 1 ? launch_typed<__half>(p, row_tiles, stream) : launch_typed<__nv_bfloat16>(p, row_tiles, stream);
}

}  // namespace msda_b200
