// Cross attention backward on the fifth-generation tensor cores, 16-bit types.
//
// One kernel template in two forms.  A CTA holds a tile X of 128 and walks tiles Y of 64:
//
//   KEYS    X = k, v      Y = q, do     dv = sum P do, dk = sum dS q
//   else    X = q, do     Y = k, v                     dq = sum dS k
//
//   S = X0 Y0^T   T = X1 Y1^T   P = exp2(c S - L)   dS = P (T - delta)
//   acc0 += P Y1 (KEYS)         acc1 += dS Y0
//
// Either way a thread owns a row of S and T (a lane of tensor memory), P and dS go back to tensor
// memory in 16 bits as left operands, and the walked tile serves both products from one copy in shared
// memory (rows along k, then rows along the other axis).  The weights are formed twice, in both
// forms, so that every gradient is summed by one CTA in one order: no atomics.  Two warpgroups take
// the Y tiles in turn, each with scores of its own; a CTA goes on to the next X tile while the sums of
// the last one are written.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace msda_b200 {

namespace {

constexpr int kX = 128, kY = 64;

template <int DP>
constexpr int kStages = DP == 128 ? 2 : 4;

template <int DP, bool KEYS>
struct Shared {
    static constexpr int ST = kStages<DP>;
    alignas(1024) unsigned char x[2][2][kX * DP * 2];          // two items' X0 and X1
    alignas(1024) unsigned char y[ST][2][kY * DP * 2];
    alignas(16) float lse[KEYS ? ST : 1][kY];                   // of the walked rows, both with the sign turned
    alignas(16) float delta[KEYS ? ST : 1][kY];
    alignas(16) uint32_t words[KEYS ? ST : 1][4][kY];           // word w of a row: states 32 w .. of X
    uint64_t x_full[2], x_free[2], y_full[ST], y_free[ST], row_full[ST], row_free[ST];
    uint64_t s_full[2], p_full[2], acc_full, acc_free;
    uint32_t tmem;
};

struct Item {
    int first, part, b, h, begin, end;       // of X; of Y, in tiles
    int64_t bh;
};

// x_rows, y_rows: rows that a tile takes (all of them for states; whole groups of heads for packed rows)
template <bool KEYS>
__device__ __forceinline__ Item item_of(const AttentionParams &p, int64_t i, int x_rows, int y_rows) {
    const int X = KEYS ? p.S : p.R, Y = KEYS ? p.R : p.S;
    const int x_tiles = (X + x_rows - 1) / x_rows, y_tiles = (Y + y_rows - 1) / y_rows;
    Item t;
    t.first = (int)(i % x_tiles) * x_rows;
    i /= x_tiles;
    t.part = (int)(i % p.splits);
    t.bh = i / p.splits;
    t.b = (int)(t.bh / p.K), t.h = (int)(t.bh % p.K);
    t.begin = t.part * p.tiles;
    t.end = min(y_tiles, t.begin + p.tiles);
    if constexpr (KEYS) {
        const uint32_t *words = key_words_of(p, t.b, t.h);
        if (words != nullptr) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(words + t.first / 32));
            if ((w.x | w.y | w.z | w.w) == 0) t.end = t.begin;              // nobody sees these states
        }
    }
    return t;
}

// the first tile of 64 states from t on in which some may be seen
__device__ __forceinline__ int next_tile(const uint32_t *words, int t, int end) {
    if (words == nullptr) return t;
    for (; t < end; ++t) {
        const uint2 w = __ldg(reinterpret_cast<const uint2 *>(words) + t);
        if (w.x | w.y) return t;
    }
    return end;
}

// 64 columns of exponents or differences at a time: x = a * scale + b over pairs
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    ffma2(c, a, b);
    return c;
}

template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(384, 1)
    attention_backward_tc_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ tc::TensorMap x0m,
                                 const __grid_constant__ tc::TensorMap x1m, const __grid_constant__ tc::TensorMap y0m,
                                 const __grid_constant__ tc::TensorMap y1m, int64_t items, int x_rows, int y_rows) {
    using namespace tc;
    constexpr int ST = kStages<DP>;
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr uint32_t kS = 0, kT = 64, kGroup = 128, kAcc0 = 256, kAcc1 = KEYS ? 256 + DP : 256;
    extern __shared__ __align__(1024) unsigned char raw[];
    auto &sm = *reinterpret_cast<Shared<DP, KEYS> *>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 8) tmem_alloc(&sm.tmem, 512);
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            barrier_init(&sm.x_full[s], 1), barrier_init(&sm.x_free[s], 1);
            barrier_init(&sm.s_full[s], 1), barrier_init(&sm.p_full[s], 128);
        }
        for (int s = 0; s < ST; ++s) {
            barrier_init(&sm.y_full[s], 1), barrier_init(&sm.y_free[s], 1);
            barrier_init(&sm.row_full[s], 32), barrier_init(&sm.row_free[s], 128);
        }
        barrier_init(&sm.acc_full, 1), barrier_init(&sm.acc_free, 256);
    }
    if (y_rows < kY) {      // rows that no load reaches
        for (int i = threadIdx.x; i < (int)sizeof(sm.y) / 16; i += 384) reinterpret_cast<uint4 *>(sm.y)[i] = make_uint4(0, 0, 0, 0);
        fence_async_shared();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm.tmem;
    bool fine = true;

    if (warp < 8) {
        registers_up<224>();
        const int group = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t mine = tmem + group * kGroup + lanes;
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
        int n = 0, done = 0;             // tiles and items with tiles so far
        for (int64_t i = blockIdx.x; fine && i < items; i += gridDim.x) {
            const Item it = item_of<KEYS>(p, i, x_rows, y_rows);
            const uint32_t *words = key_words_of(p, it.b, it.h);
            const int x = it.first + row;
            const bool mine_valid = row < x_rows && x < (KEYS ? p.S : p.R);
            const bool idle = (row & ~31) >= x_rows || it.first + (row & ~31) >= (KEYS ? p.S : p.R);
            float my_lse = -INFINITY, my_delta = 0.f;
            const uint32_t *rw = nullptr;
            bool seen = false;
            if constexpr (KEYS) {
                seen = mine_valid && ((key_word(words, p.S, x >> 5) >> (x & 31)) & 1);
            } else if (mine_valid) {
                my_lse = -p.lse[it.bh * p.R + x];
                my_delta = -p.delta[it.bh * p.R + x];
                rw = row_words_of(p, it.b, it.h, x);
            }
            const int before = n;
            for (int tile = KEYS ? it.begin : next_tile(words, it.begin, it.end); fine && tile < it.end; ++n) {
                const int next = KEYS ? tile + 1 : next_tile(words, tile + 1, it.end);
                if ((n & 1) != group) {
                    tile = next;
                    continue;
                }
                const int stage = n % ST;
                uint2 see = make_uint2(0, 0);
                if constexpr (!KEYS)
                    see = rw != nullptr ? __ldg(reinterpret_cast<const uint2 *>(rw) + tile)
                                        : make_uint2(key_word(words, p.S, 2 * tile), key_word(words, p.S, 2 * tile + 1));
                if constexpr (KEYS) fine = barrier_wait(&sm.row_full[stage], (n / ST) & 1);
                fine = barrier_wait(&sm.s_full[group], (n >> 1) & 1) && fine;
                if (!fine) break;
                fence_after();
                if (!idle) {
                    uint32_t s[2][32], t[2][32];
                    tmem_load32(s[0], mine + kS), tmem_load32(s[1], mine + kS + 32);
                    tmem_wait_load();
                    loaded(s[0]), loaded(s[1]);
                    tmem_load32(t[0], mine + kT), tmem_load32(t[1], mine + kT + 32);
                    float2 w[32];
                    uint32_t packed[32];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const uint32_t *from = &s[c >> 4][(2 * c) & 31];
                        float4 l = make_float4(my_lse, my_lse, my_lse, my_lse);
                        if constexpr (KEYS) l = *reinterpret_cast<const float4 *>(&sm.lse[stage][2 * c]);
                        w[c] = fma2(make_float2(__uint_as_float(from[0]), __uint_as_float(from[1])), scale2, make_float2(l.x, l.y));
                        w[c + 1] = fma2(make_float2(__uint_as_float(from[2]), __uint_as_float(from[3])), scale2, make_float2(l.z, l.w));
                        w[c].x = fast_exp2(w[c].x), w[c].y = fast_exp2(w[c].y);
                        w[c + 1].x = fast_exp2(w[c + 1].x), w[c + 1].y = fast_exp2(w[c + 1].y);
                    }
                    // which of the 64 may be seen; `some` where not all of the warp's are
                    const bool some = KEYS ? p.row_words != nullptr || !__all_sync(0xffffffffu, seen)
                                           : !__all_sync(0xffffffffu, (see.x & see.y) == 0xffffffffu);
                    uint32_t see0 = see.x, see1 = see.y;
                    if (some) {
                        if constexpr (KEYS) {
                            see0 = see1 = seen ? 0xffffffffu : 0u;
                            if (p.row_words != nullptr) {
                                see0 = see1 = 0;
                                const uint32_t *of = sm.words[stage][warp & 3];
#pragma unroll
                                for (int c = 0; c < 32; ++c) {
                                    see0 |= ((of[c] >> lane) & 1u) << c;
                                    see1 |= ((of[32 + c] >> lane) & 1u) << c;
                                }
                            }
                        }
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            const uint32_t bits = c < 16 ? see0 >> (2 * c) : see1 >> (2 * c - 32);
                            if (!(bits & 1)) w[c].x = 0.f;
                            if (!(bits & 2)) w[c].y = 0.f;
                        }
                    }
                    if constexpr (KEYS) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) packed[c] = VecTraits<T>::pack2(w[c]);
                        tmem_store32(mine + kS, packed);
                    }
                    tmem_wait_load();
                    loaded(t[0]), loaded(t[1]);
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const uint32_t *from = &t[c >> 4][(2 * c) & 31];
                        float4 d = make_float4(my_delta, my_delta, my_delta, my_delta);
                        if constexpr (KEYS) d = *reinterpret_cast<const float4 *>(&sm.delta[stage][2 * c]);
                        const float2 one = make_float2(1.f, 1.f);
                        w[c] = fmul2(w[c], fma2(make_float2(__uint_as_float(from[0]), __uint_as_float(from[1])), one, make_float2(d.x, d.y)));
                        w[c + 1] = fmul2(w[c + 1], fma2(make_float2(__uint_as_float(from[2]), __uint_as_float(from[3])), one, make_float2(d.z, d.w)));
                    }
                    if (some) {
                        // (0 times what an unseen state's v holds)
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            const uint32_t bits = c < 16 ? see0 >> (2 * c) : see1 >> (2 * c - 32);
                            if (!(bits & 1)) w[c].x = 0.f;
                            if (!(bits & 2)) w[c].y = 0.f;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 32; ++c) packed[c] = VecTraits<T>::pack2(w[c]);
                    tmem_store32(mine + kT, packed);
                    tmem_wait_store();
                }
                if constexpr (KEYS) barrier_arrive(&sm.row_free[stage]);
                fence_before();
                barrier_arrive(&sm.p_full[group]);
                tile = next;
            }
            const bool some = n > before;
            if (some) {
                fine = fine && barrier_wait(&sm.acc_full, done & 1);
                fence_after();
                ++done;
            }
            // sums to memory: each group takes one of the two, or half of the one
            constexpr int kHalf = KEYS ? DP : DP / 2;
            const uint32_t acc = tmem + lanes + (KEYS ? (group == 0 ? kAcc0 : kAcc1) : kAcc1 + group * kHalf);
            const int from = KEYS ? 0 : group * kHalf;
            const float factor = !fine ? NAN : KEYS && group == 0 ? 1.f : p.scale;
            const int rows = KEYS ? p.S : p.R;
            const int query = x / p.share;
            const int64_t at = KEYS ? (((int64_t)it.b * p.S + x) * p.K + it.h) * p.D
                                    : (((int64_t)it.b * p.Q + query) * p.K * p.share + it.h * p.share + (x - query * p.share)) * p.D;
            T *out = static_cast<T *>(KEYS ? (group == 0 ? p.dv : p.dk) : p.dq) + at;
            float *parts = (KEYS && group == 0 ? p.part2 : p.part) +
                           ((it.part * (int64_t)p.B * p.K + it.bh) * rows + x) * p.D;
#pragma unroll
            for (int d = 0; d < kHalf; d += 16) {
                uint32_t v[16];
                if (some && !idle) {
                    tmem_load16(v, acc + d);
                    tmem_wait_load();
                    loaded(v);
                }
                float2 y[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    y[c] = some ? make_float2(__uint_as_float(v[2 * c]) * factor, __uint_as_float(v[2 * c + 1]) * factor)
                                : make_float2(0.f, 0.f);
                if (!mine_valid) continue;
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const int col = from + d + 2 * c;
                    if (col >= p.D) continue;
                    if (p.splits > 1) {
                        *reinterpret_cast<float4 *>(parts + col) = make_float4(y[c].x, y[c].y, y[c + 1].x, y[c + 1].y);
                        *reinterpret_cast<float4 *>(parts + col + 4) = make_float4(y[c + 2].x, y[c + 2].y, y[c + 3].x, y[c + 3].y);
                    } else {
                        const float2 z[4] = {y[c], y[c + 1], y[c + 2], y[c + 3]};
                        *reinterpret_cast<uint4 *>(out + col) = VecTraits<T>::pack(z);
                    }
                }
            }
            if (some) {
                fence_before();
                barrier_arrive(&sm.acc_free);
            }
        }
    } else {
        registers_down<56>();
        if (warp == 8 && lane == 0) {
            int n = 0, done = 0;
            for (int64_t i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of<KEYS>(p, i, x_rows, y_rows);
                const uint32_t *words = key_words_of(p, it.b, it.h);
                int tile = KEYS ? it.begin : next_tile(words, it.begin, it.end);
                if (tile >= it.end) continue;
                const int buffer = done & 1;
                if (done > 1) fine = barrier_wait(&sm.x_free[buffer], ((done >> 1) - 1) & 1);
                if (!fine) break;
                barrier_expect(&sm.x_full[buffer], 2 * x_rows * DP * 2);
                load_rows<DP, kX>(sm.x[buffer][0], x0m, &sm.x_full[buffer], it.b, it.h, it.first);
                load_rows<DP, kX>(sm.x[buffer][1], x1m, &sm.x_full[buffer], it.b, it.h, it.first);
                ++done;
                for (; fine && tile < it.end; ++n) {
                    const int stage = n % ST;
                    if (n >= ST) fine = barrier_wait(&sm.y_free[stage], (n / ST - 1) & 1);
                    if (!fine) break;
                    barrier_expect(&sm.y_full[stage], 2 * y_rows * DP * 2);
                    load_rows<DP, kY>(sm.y[stage][0], y0m, &sm.y_full[stage], it.b, it.h, tile * y_rows);
                    load_rows<DP, kY>(sm.y[stage][1], y1m, &sm.y_full[stage], it.b, it.h, tile * y_rows);
                    tile = KEYS ? tile + 1 : next_tile(words, tile + 1, it.end);
                }
            }
            if (!fine) {     // nothing may still be on its way when the CTA ends
                for (int s = 0; s < 2; ++s)
                    if (done > s) barrier_wait(&sm.x_full[s], ((done - s + 1) / 2 - 1) & 1);
                for (int s = 0; s < ST; ++s)
                    if (n > s) barrier_wait(&sm.y_full[s], ((n - s + ST - 1) / ST - 1) & 1);
            }
        } else if (warp == 10 && KEYS) {
            // what the walked rows need beside their tiles
            int n = 0;
            for (int64_t i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of<KEYS>(p, i, x_rows, y_rows);
                for (int tile = it.begin; fine && tile < it.end; ++tile, ++n) {
                    const int stage = n % ST;
                    float lse[2], delta[2];
                    uint4 see[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = lane + 32 * c, r = tile * y_rows + col;
                        const bool valid = col < y_rows && r < p.R;
                        lse[c] = valid ? -p.lse[it.bh * p.R + r] : -INFINITY;
                        delta[c] = valid ? -p.delta[it.bh * p.R + r] : 0.f;
                        if (p.row_words != nullptr)
                            see[c] = valid ? __ldg(reinterpret_cast<const uint4 *>(row_words_of(p, it.b, it.h, r) + it.first / 32))
                                           : make_uint4(0, 0, 0, 0);
                    }
                    if (n >= ST) fine = barrier_wait(&sm.row_free[stage], (n / ST - 1) & 1);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = lane + 32 * c;
                        sm.lse[stage][col] = lse[c];
                        sm.delta[stage][col] = delta[c];
                        if (p.row_words != nullptr) {
                            sm.words[stage][0][col] = see[c].x, sm.words[stage][1][col] = see[c].y;
                            sm.words[stage][2][col] = see[c].z, sm.words[stage][3][col] = see[c].w;
                        }
                    }
                    barrier_arrive(&sm.row_full[stage]);
                }
            }
        } else if (warp == 9) {
            constexpr uint32_t kScores = instruction(kBf16, kX, kY, false, false);
            constexpr uint32_t kSums = instruction(kBf16, kX, DP, false, true);
            constexpr int kRow = kRowBytes<DP>;
            // the tile whose products with P and dS are still to be issued
            int pending = -1, pending_n = 0;
            bool pending_first = false;
            const uint32_t *pending_words = nullptr;
            int n = 0, done = 0;
            const auto issue_sums = [&](bool last) {
                const int group = pending_n & 1, stage = pending_n % ST;
                if (pending_first && done > 1) fine = fine && barrier_wait(&sm.acc_free, (done - 2) & 1);
                fine = fine && barrier_wait(&sm.p_full[group], (pending_n >> 1) & 1);
                if (!KEYS && pending_words != nullptr && fine) {
                    // rows of k that nobody may see: their dS is 0 and its products have to be
                    const uint2 see = __ldg(reinterpret_cast<const uint2 *>(pending_words) + pending);
                    if ((see.x & see.y) != 0xffffffffu) {
                        constexpr int kChunks = DP / 8;
                        for (int c = lane; c < 64 * kChunks; c += 32) {
                            const int r = c / kChunks;
                            if (!(((r < 32 ? see.x : see.y) >> (r & 31)) & 1))
                                *reinterpret_cast<uint4 *>(sm.y[stage][0] + swizzled<DP, kY>(r, c % kChunks)) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_shared();
                        __syncwarp();
                    }
                }
                fence_after();
                if (fine && lane == 0) {
                    const uint32_t from = tmem + group * kGroup;
                    const uint32_t y0 = smem_address(sm.y[stage][0]), y1 = smem_address(sm.y[stage][1]);
                    if constexpr (KEYS)
#pragma unroll
                        for (int j = 0; j < kY; j += 16)
                            mma_ts(tmem + kAcc0, from + kS + j / 2, descriptor<kRow>(y1 + j * kRow, kY * 128), kSums, !pending_first || j > 0);
#pragma unroll
                    for (int j = 0; j < kY; j += 16)
                        mma_ts(tmem + kAcc1, from + kT + j / 2, descriptor<kRow>(y0 + j * kRow, kY * 128), kSums, !pending_first || j > 0);
                    commit(&sm.y_free[stage]);
                    if (last) commit(&sm.acc_full);
                }
                pending = -1;
            };
            for (int64_t i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of<KEYS>(p, i, x_rows, y_rows);
                const uint32_t *words = key_words_of(p, it.b, it.h);
                int tile = KEYS ? it.begin : next_tile(words, it.begin, it.end);
                if (tile >= it.end) continue;
                const int buffer = done & 1;
                fine = barrier_wait(&sm.x_full[buffer], (done >> 1) & 1);
                bool first = true;
                for (; fine && tile < it.end; ++n) {
                    const int next = KEYS ? tile + 1 : next_tile(words, tile + 1, it.end);
                    const int stage = n % ST, group = n & 1;
                    fine = barrier_wait(&sm.y_full[stage], (n / ST) & 1);
                    fence_after();
                    if (fine && lane == 0) {
                        const uint32_t to = tmem + group * kGroup;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t xa = smem_address(sm.x[buffer][half]), ya = smem_address(sm.y[stage][half]);
#pragma unroll
                            for (int d = 0; d < DP; d += 16)
                                mma(to + (half == 0 ? kS : kT), descriptor<kRow>(xa + (d >> 6) * kX * 128 + (d & 63) * 2, 16),
                                    descriptor<kRow>(ya + (d >> 6) * kY * 128 + (d & 63) * 2, 16), kScores, d > 0);
                        }
                        commit(&sm.s_full[group]);
                        if (next >= it.end) commit(&sm.x_free[buffer]);
                    }
                    if (pending >= 0) issue_sums(first);
                    if (first) ++done;
                    pending = tile, pending_n = n, pending_first = first, pending_words = words;
                    first = false;
                    tile = next;
                }
            }
            if (pending >= 0) issue_sums(true);
        }
    }
    __syncthreads();
    if (warp == 8) {
        fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int DP, bool KEYS>
cudaError_t launch(const AttentionParams &p, cudaStream_t stream) {
    const int64_t gs[3] = {(int64_t)p.Q * p.K * p.share * p.D, (int64_t)p.K * p.share * p.D, p.D};
    const int row_tile = KEYS ? kY : kX, state_tile = KEYS ? kX : kY;
    tc::TensorMap q, g, k, v;
    if (!tc::make_map<T, DP>(q, p.q, p.qs, p.B, p.Q, p.K, p.share, p.D, row_tile) ||
        !tc::make_map<T, DP>(g, p.grad_out, gs, p.B, p.Q, p.K, p.share, p.D, row_tile) ||
        !tc::make_map<T, DP>(k, p.k, p.ks, p.B, p.S, p.K, 1, p.D, state_tile) ||
        !tc::make_map<T, DP>(v, p.v, p.vs, p.B, p.S, p.K, 1, p.D, state_tile))
        return cudaErrorNotSupported;
    const auto kernel = attention_backward_tc_kernel<T, DP, KEYS>;
    constexpr size_t smem = sizeof(Shared<DP, KEYS>);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int rows = row_tile / p.share * p.share;
    const int x_rows = KEYS ? kX : rows, y_rows = KEYS ? rows : kY;
    const int64_t items = (int64_t)p.B * p.K * p.splits * (((KEYS ? p.S : p.R) + x_rows - 1) / x_rows);
    const unsigned grid = (unsigned)std::min<int64_t>(items, 148);
    kernel<<<grid, 384, smem, stream>>>(p, KEYS ? k : q, KEYS ? v : g, KEYS ? q : k, KEYS ? g : v, items, x_rows, y_rows);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, bool keys, cudaStream_t stream) {
    if (p.D <= 32) return keys ? launch<T, 32, true>(p, stream) : launch<T, 32, false>(p, stream);
    if (p.D <= 64) return keys ? launch<T, 64, true>(p, stream) : launch<T, 64, false>(p, stream);
    return keys ? launch<T, 128, true>(p, stream) : launch<T, 128, false>(p, stream);
}

}  // namespace

cudaError_t launch_attention_backward_tc(const AttentionParams &p, int dtype, bool keys, cudaStream_t stream) {
    return dtype == 1 ? launch_typed<__half>(p, keys, stream) : launch_typed<__nv_bfloat16>(p, keys, stream);
}

}  // namespace msda_b200
