// Cross attention backward on the fifth-generation tensor cores, 16-bit types, and float32 up to 64 channels as three
// bf16 terms of every operand (TERMS = 3: six products for one).
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
// memory (rows along k, then rows along the other axis).  (16-bit types: rounded to the type that both operands of a product
// have, half a step each, and delta is that of the rounded result: gradients in bf16 2.4e-3 off, a plain form 1.7e-3.
// attn_common.cuh says what float16 is scaled by.)  The weights are formed twice, in both
// forms, so that every gradient is summed by one CTA in one order: no atomics.  Two or three warpgroups take
// the Y tiles in turn, each with scores of its own; a CTA goes on to the next X tile while the sums of
// the last one are written by a warpgroup of their own.
//
// Bound by the cycle of a warpgroup (scores, exponentials, weights back) where heads are small, by that and the tensor
// cores in turn where they are large.  4 x 300 queries over 17 821 states, 8 heads of 32, bf16: 141 us with states
// held and 109 with rows held (exponential unit 36 and 41 %, issue slots 47 %, tensor cores 16 and 18 %; half of the
// exponentials left out: 15 % less); 2 x 2048 over 4096, 16 heads on 4 of 128: 270 and 225 us (tensor cores 63 and 57 %).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace msda_b200 {

namespace {

constexpr int kX = 128, kY = 64;

template <int DP, bool KEYS, int TERMS>
struct Shape {
    static constexpr int ST = TERMS == 3 ? (DP == 32 ? 4 : 2) : DP == 128 ? 4 : 6;      // tiles Y in flight
    static constexpr int XB = DP * TERMS > 96 ? 1 : 2;                                   // tiles X
    // warpgroups that take the tiles Y in turn: as many as tensor memory has room for
    static constexpr int kGroups = TERMS == 3 || DP == 128 ? 2 : 3;
    static constexpr int kThreads = kGroups * 128 + 256;
    // what a thread may hold: all of the block's at launch, shared out anew
    static constexpr int kWriting = TERMS == 1 ? 64 : KEYS && DP == 64 ? 168 : 104;
    static constexpr int kRegisters = kGroups == 3 ? 120 : kWriting == 64 ? 192 : kWriting == 104 ? 176 : 144, kFew = 56;
    // tiles after which the writers take the sums on: those of the tensor cores are cut off, not rounded, at every
    // product that is added (2^-25.7 of the sum each, 24 times a tile with terms): over 32 tiles gradients were 1.4e-5
    // off, with runs of eight 3.3e-6, of four 1.6e-6, in the same time
    static constexpr int kRun = TERMS == 1 ? 1 << 30 : 4;
    // columns of tensor memory: of a group S and T, in whose places P and dS come (third terms need more), then the sums
    static constexpr uint32_t kS = 0, kT = 64;
    __host__ __device__ static constexpr uint32_t third(bool p) { return KEYS && !p ? 160 : 128; }
    static constexpr uint32_t kGroup = TERMS == 1 ? 128 : KEYS ? 192 : 160;
    static constexpr uint32_t kAcc = kGroups * kGroup, kSums = KEYS ? 2 * DP : DP;      // dv and dk, or dq
    static constexpr int AB = kAcc + 2 * kSums <= 512 ? 2 : 1;                           // of as many items
    static_assert(kAcc + AB * kSums <= 512);
    static_assert(ST >= kGroups);
};

template <int DP, bool KEYS, int TERMS>
struct Shared {
    using Sh = Shape<DP, KEYS, TERMS>;
    static constexpr int ST = Sh::ST;
    alignas(1024) unsigned char x[Sh::XB][2][TERMS][kX * DP * 2];       // of an item X0 and X1
    alignas(1024) unsigned char y[ST][2][TERMS][kY * DP * 2];
    alignas(16) float lse[KEYS ? ST : 1][kY];                   // of the walked rows, both with the sign turned
    alignas(16) float delta[KEYS ? ST : 1][kY];
    alignas(16) uint32_t words[KEYS ? ST : 1][4][kY];           // word w of a row: states 32 w .. of X
    uint64_t x_full[2], x_free[2], y_full[ST], y_free[ST], y_clean[ST], row_full[ST], row_free[ST];
    uint64_t s_full[Sh::kGroups], p_full[Sh::kGroups], acc_full[2], acc_free[2];
    uint32_t tmem;
};

// What a CTA does at a time: a tile X and a stretch of tiles Y.
struct Item {
    int first, part, b, h;       // of X
    int64_t bh;
};

// x_rows: rows that a tile takes (all of them for states; whole groups of heads for packed rows)
__device__ __forceinline__ Item item_of(const AttentionParams &p, unsigned i, unsigned x_tiles, int x_rows) {
    Item t;
    const unsigned j = i / x_tiles, bh = j / p.splits;
    t.first = (int)(i - j * x_tiles) * x_rows;
    t.part = (int)(j - bh * p.splits);
    t.bh = bh;
    t.b = (int)(bh / p.K), t.h = (int)(bh - t.b * p.K);
    return t;
}

// the tiles Y of an item: listed tiles of states, or all of the rows
template <bool KEYS>
struct Walk;
template <>
struct Walk<false> : Tiles<kY> {
    __device__ __forceinline__ Walk(const AttentionParams &p, const Item &t, int) : Tiles<kY>(p, t.b, t.h, t.part) {}
};
template <>
struct Walk<true> {
    int first, count;
    __device__ __forceinline__ Walk(const AttentionParams &p, const Item &t, int y_rows) {
        const int all = (p.R + y_rows - 1) / y_rows;
        Tiles<kY>::stretch(all, p.splits, t.part, first, count);
        const uint32_t *words = key_words_of(p, t.b, t.h);
        if (words != nullptr) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(words + t.first / 32));
            if ((w.x | w.y | w.z | w.w) == 0) count = 0;                  // nobody sees these states
        }
    }
    __device__ __forceinline__ uint32_t operator[](int n) const { return (uint32_t)(first + n); }
};

template <typename T, int DP, bool KEYS, int TERMS>
__global__ void __launch_bounds__(Shape<DP, KEYS, TERMS>::kThreads, 1)
    attention_backward_tc_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ tc::TensorMap x0m,
                                 const __grid_constant__ tc::TensorMap x1m, const __grid_constant__ tc::TensorMap y0m,
                                 const __grid_constant__ tc::TensorMap y1m, unsigned items, int x_rows, int y_rows) {
    using namespace tc;
    using Sh = Shape<DP, KEYS, TERMS>;
    using Out = std::conditional_t<TERMS == 3, float, T>;      // of the call's tensors; T is that of the products
    constexpr int ST = Sh::ST, XB = Sh::XB, kGroups = Sh::kGroups, kLast = 4 * kGroups, kWriters = kLast + 4;
    constexpr int kPairsOf = TERMS == 3 ? kPairs : 1;
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr int AB = Sh::AB;
    constexpr uint32_t kS = Sh::kS, kT = Sh::kT, kGroup = Sh::kGroup;
    constexpr uint32_t kXBytes = kX * DP * 2, kYBytes = kY * DP * 2;
    extern __shared__ __align__(1024) unsigned char raw[];
    auto &sm = *reinterpret_cast<Shared<DP, KEYS, TERMS> *>(raw);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (warp == kLast) tmem_alloc(&sm.tmem, 512);
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            barrier_init(&sm.x_full[s], 1), barrier_init(&sm.x_free[s], 1);
        }
        for (int g = 0; g < kGroups; ++g) barrier_init(&sm.s_full[g], 1), barrier_init(&sm.p_full[g], 128);
        for (int s = 0; s < ST; ++s) {
            barrier_init(&sm.y_full[s], 1), barrier_init(&sm.y_free[s], 1);
            barrier_init(&sm.y_clean[s], 32);
            barrier_init(&sm.row_full[s], 32), barrier_init(&sm.row_free[s], 128);
        }
        for (int s = 0; s < 2; ++s) barrier_init(&sm.acc_full[s], 1), barrier_init(&sm.acc_free[s], 128);
        fence_async_shared();
    }
    if (y_rows < kY) {      // rows that no load reaches
        for (int i = threadIdx.x; i < (int)sizeof(sm.y) / 16; i += Sh::kThreads) reinterpret_cast<uint4 *>(sm.y)[i] = make_uint4(0, 0, 0, 0);
        fence_async_shared();
    }
    grid_dependency_wait();            // (of what this call has launched before)
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    const unsigned x_tiles = ((KEYS ? p.S : p.R) + x_rows - 1) / x_rows;
    bool fine = true;

    if (warp < kLast) {
        registers_up<Sh::kRegisters>();
        const int group = warp >> 2, row = threadIdx.x & 127;
        const uint32_t mine = tmem + group * kGroup + ((uint32_t)(warp & 3) << 21);
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
        const bool own_words = p.row_words != nullptr;
        const auto put = [](float2 x, uint32_t (&to)[TERMS][16], int c) {
            if constexpr (TERMS == 3) {
                uint32_t t[3];
                split_terms(x, t);
                to[0][c] = t[0], to[1][c] = t[1], to[TERMS - 1][c] = t[2];
            } else {
                to[0][c] = VecTraits<T>::pack2(x);
            }
        };
        int before = 0, n = group;       // tiles of the items so far; this group's next one
        Ring<ST> y;
        uint32_t turn = 0;               // parity of the group's tiles
        y.next(group);
        for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
            const Item it = item_of(p, i, x_tiles, x_rows);
            const Walk<KEYS> walk(p, it, y_rows);
            const uint32_t *words = key_words_of(p, it.b, it.h);
            const int x = it.first + row;
            const bool mine_valid = row < x_rows && x < (KEYS ? p.S : p.R);
            const bool idle = (row & ~31) >= x_rows || it.first + (row & ~31) >= (KEYS ? p.S : p.R);
            float my_lse = -INFINITY, my_delta = 0.f;
            [[maybe_unused]] float grow = 1.f;           // float16: what dS is scaled by, less what P is by
            const uint32_t *rw = nullptr;
            bool seen = false;
            if constexpr (KEYS) {
                seen = mine_valid && ((key_word(words, p.S, x >> 5) >> (x & 31)) & 1);
                if (kScaled<T> && mine_valid) grow = state_scale(p, it.bh, x) * (1.f / kWeightScale);
            } else if (mine_valid) {
                my_lse = -p.lse[it.bh * p.R + x];
                if constexpr (kScaled<T>) grow = row_scale(p, it.bh, x);
                my_delta = -p.delta[it.bh * p.R + x] * grow;
                rw = row_words_of(p, it.b, it.h, x);
            }
            if (rw == nullptr) rw = words;
            // T - delta, scaled (rows held: delta is already)
            const auto less = [&](float2 t, float2 d) {
                if constexpr (!kScaled<T>) return add2(t, d);
                else if constexpr (KEYS) return fmul2(add2(t, d), make_float2(grow, grow));
                else return fma2(t, make_float2(grow, grow), d);
            };
            uint32_t entry = 0;
            uint2 see = make_uint2(0, 0);
            // the mask of this group's next tile comes while it works on another
            const auto fetch = [&](int at) {
                if (at >= before + walk.count) return;
                entry = walk[at - before];
                if (rw != nullptr && (own_words || !(entry >> 31)))
                    see = __ldg(reinterpret_cast<const uint2 *>(rw) + (entry & 0x7fffffff));
            };
            if constexpr (!KEYS) fetch(n);
            for (; fine && n < before + walk.count; n += kGroups, y.next(kGroups), turn ^= 1) {
                const int stage = y.at;
                const uint32_t now = entry;
                const uint2 may = see;
                if constexpr (!KEYS) fetch(n + kGroups);
                if constexpr (KEYS) fine = barrier_wait(&sm.row_full[stage], y.parity);
                fine = barrier_wait(&sm.s_full[group], turn) && fine;
                if (!fine) break;
                fence_after();
                if (!idle) {
                    uint32_t s[32], t[32];
                    tmem_load32(s, mine + kS);
                    // which of the 64 may be seen; `some` where not all of the warp's are
                    const bool some = KEYS ? own_words || !__all_sync(0xffffffffu, seen)
                                      : own_words ? !__all_sync(0xffffffffu, (may.x & may.y) == 0xffffffffu) : !(now >> 31);
                    uint32_t sees[2] = {may.x, may.y};
                    if (some) {
                        if constexpr (KEYS) {
                            sees[0] = sees[1] = seen ? 0xffffffffu : 0u;
                            if (own_words) {
                                const uint32_t *of = sm.words[stage][warp & 3];
                                sees[0] = sees[1] = 0;
#pragma unroll
                                for (int c = 0; c < 32; ++c) {
                                    sees[0] |= ((of[c] >> lane) & 1u) << c;
                                    sees[1] |= ((of[32 + c] >> lane) & 1u) << c;
                                }
                            }
                        } else if (rw == nullptr) {
                            sees[0] = key_word(nullptr, p.S, 2 * (now & 0x7fffffff));
                            sees[1] = key_word(nullptr, p.S, 2 * (now & 0x7fffffff) + 1);
                        }
                    }
                    // Half by half, loads under the work on what came before.  What is stored takes the place of
                    // columns that are in registers by then: P that of S's first half, dS that of T's; their second
                    // terms would take the second halves, and wait for those.
                    uint32_t second[TERMS == 3 ? 16 : 1], later[TERMS == 3 ? 16 : 1];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        tmem_wait_load();
                        loaded(s);
                        tmem_load32(t, mine + kT + 32 * half);
                        float2 w[16];
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float4 l = make_float4(my_lse, my_lse, my_lse, my_lse);
                            if constexpr (KEYS) l = *reinterpret_cast<const float4 *>(&sm.lse[stage][32 * half + 2 * c]);
                            w[c] = fma2(make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, make_float2(l.x, l.y));
                            w[c + 1] = fma2(make_float2(__uint_as_float(s[2 * c + 2]), __uint_as_float(s[2 * c + 3])), scale2, make_float2(l.z, l.w));
                            w[c].x = fast_exp2(w[c].x), w[c].y = fast_exp2(w[c].y);
                            w[c + 1].x = fast_exp2(w[c + 1].x), w[c + 1].y = fast_exp2(w[c + 1].y);
                        }
                        if (some) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                if (!((sees[half] >> (2 * c)) & 1)) w[c].x = 0.f;
                                if (!((sees[half] >> (2 * c)) & 2)) w[c].y = 0.f;
                            }
                        }
                        uint32_t packed[TERMS][16];
                        if constexpr (KEYS) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) put(w[c], packed, c);
                            if constexpr (TERMS == 3) {
                                if (half == 0) {
#pragma unroll
                                    for (int c = 0; c < 16; ++c) second[c] = packed[1][c];
                                } else {
                                    tmem_store16(mine + kS + 32, second);
                                    tmem_store16(mine + kS + 48, packed[1]);
                                }
                                tmem_store16(mine + Sh::third(true) + 16 * half, packed[TERMS - 1]);
                            }
                            tmem_store16(mine + kS + 16 * half, packed[0]);
                        }
                        tmem_wait_load();
                        loaded(t);
                        if (half == 0) tmem_load32(s, mine + kS + 32);
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float4 d = make_float4(my_delta, my_delta, my_delta, my_delta);
                            if constexpr (KEYS) d = *reinterpret_cast<const float4 *>(&sm.delta[stage][32 * half + 2 * c]);
                            w[c] = fmul2(w[c], less(make_float2(__uint_as_float(t[2 * c]), __uint_as_float(t[2 * c + 1])), make_float2(d.x, d.y)));
                            w[c + 1] = fmul2(w[c + 1], less(make_float2(__uint_as_float(t[2 * c + 2]), __uint_as_float(t[2 * c + 3])), make_float2(d.z, d.w)));
                        }
                        if (some) {
                            // (0 times what an unseen state's v holds)
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                if (!((sees[half] >> (2 * c)) & 1)) w[c].x = 0.f;
                                if (!((sees[half] >> (2 * c)) & 2)) w[c].y = 0.f;
                            }
                        }
#pragma unroll
                        for (int c = 0; c < 16; ++c) put(w[c], packed, c);
                        tmem_store16(mine + kT + 16 * half, packed[0]);
                        if constexpr (TERMS == 3) {
                            tmem_store16(mine + Sh::third(false) + 16 * half, packed[TERMS - 1]);
                            if (half == 0) {
#pragma unroll
                                for (int c = 0; c < 16; ++c) later[c] = packed[1][c];
                            } else {
                                tmem_store16(mine + kT + 32, later);
                                tmem_store16(mine + kT + 48, packed[1]);
                            }
                        }
                    }
                    tmem_wait_store();
                }
                if constexpr (KEYS) barrier_arrive(&sm.row_free[stage]);
                fence_before();
                barrier_arrive(&sm.p_full[group]);
            }
            before += walk.count;
        }
    } else if (warp >= kWriters) {
        // sums to memory, while the next item is worked on
        if constexpr (Sh::kWriting > 128) registers_up<Sh::kWriting>(); else registers_down<Sh::kWriting>();
        const int row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        Ring<AB> sums;
        for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
            const Item it = item_of(p, i, x_tiles, x_rows);
            const Walk<KEYS> walk(p, it, y_rows);
            const int rows = KEYS ? p.S : p.R, x = it.first + row;
            const bool valid = row < x_rows && x < rows;
            const bool idle = (row & ~31) >= x_rows || it.first + (row & ~31) >= rows;
            float unscale = p.scale;                  // of dk and dq
            if (kScaled<T> && valid) unscale /= KEYS ? state_scale(p, it.bh, x) : row_scale(p, it.bh, x);
            const int query = x / p.share;
            const int64_t at = KEYS ? (((int64_t)it.b * p.S + x) * p.K + it.h) * p.D
                                    : (((int64_t)it.b * p.Q + query) * p.K * p.share + it.h * p.share + (x - query * p.share)) * p.D;
            const int64_t part_at = ((it.part * (int64_t)p.B * p.K + it.bh) * rows + x) * p.D;
            constexpr int kOf = TERMS == 3 ? (int)Sh::kSums : 2;
            [[maybe_unused]] float sum[kOf];          // float32: of the runs so far
#pragma unroll
            for (int c = 0; c < kOf; ++c) sum[c] = 0.f;
            if constexpr (TERMS == 3) {
                for (int j = 0; j < walk.count; j += Sh::kRun, sums.next()) {
                    fine = fine && barrier_wait(&sm.acc_full[sums.at], sums.parity);
                    fence_after();
                    if (!idle) {
#pragma unroll
                        for (int d = 0; d < (int)Sh::kSums; d += 16) {
                            uint32_t v[16];
                            tmem_load16(v, tmem + lanes + Sh::kAcc + sums.at * Sh::kSums + d);
                            tmem_wait_load();
                            loaded(v);
#pragma unroll
                            for (int c = 0; c < 16; ++c) sum[d + c] += __uint_as_float(v[c]);
                        }
                    }
                    fence_before();
                    barrier_arrive(&sm.acc_free[sums.at]);
                }
            } else if (walk.count > 0) {
                fine = barrier_wait(&sm.acc_full[sums.at], sums.parity);
                fence_after();
            }
#pragma unroll
            for (int which = KEYS ? 0 : 1; which < 2; ++which) {
                constexpr int kSecond = KEYS ? DP : 0;
                const uint32_t acc = tmem + lanes + Sh::kAcc + sums.at * Sh::kSums + (which == 1 ? kSecond : 0);
                const float factor = !fine ? NAN : which == 1 ? unscale : kScaled<T> ? 1.f / kWeightScale : 1.f;
                Out *out = static_cast<Out *>(KEYS ? (which == 0 ? p.dv : p.dk) : p.dq) + at;
                float *parts = (which == 0 ? p.part2 : p.part) + part_at;
#pragma unroll
                for (int d = 0; d < DP; d += 16) {
                    float2 y[8];
                    if constexpr (TERMS == 3) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const int of = (which == 1 ? kSecond : 0) + d + 2 * c;
                            y[c] = make_float2(sum[of] * factor, sum[of + 1] * factor);
                        }
                    } else {
                        uint32_t v[16];
                        if (walk.count > 0 && !idle) {
                            tmem_load16(v, acc + d);
                            tmem_wait_load();
                            loaded(v);
                        }
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            y[c] = walk.count > 0 ? make_float2(__uint_as_float(v[2 * c]) * factor, __uint_as_float(v[2 * c + 1]) * factor)
                                                  : make_float2(0.f, 0.f);
                    }
                    if (!valid) continue;
#pragma unroll
                    for (int c = 0; c < 8; c += 4) {
                        const int col = d + 2 * c;
                        if (col >= p.D) continue;
                        if (TERMS == 3 || p.splits > 1) {
                            float *to = p.splits > 1 ? parts : reinterpret_cast<float *>(out);
                            *reinterpret_cast<float4 *>(to + col) = make_float4(y[c].x, y[c].y, y[c + 1].x, y[c + 1].y);
                            if (col + 4 < p.D)
                                *reinterpret_cast<float4 *>(to + col + 4) = make_float4(y[c + 2].x, y[c + 2].y, y[c + 3].x, y[c + 3].y);
                        } else if constexpr (TERMS == 1) {
                            const float2 z[4] = {y[c], y[c + 1], y[c + 2], y[c + 3]};
                            *reinterpret_cast<uint4 *>(out + col) = VecTraits<T>::pack(z);
                        }
                    }
                }
            }
            if (TERMS == 1 && walk.count > 0) {
                fence_before();
                barrier_arrive(&sm.acc_free[sums.at]);
                sums.next();
            }
        }
    } else {
        registers_down<Sh::kFew>();
        if (warp == kLast && elect_one()) {
            int n = 0, done = 0;
            Ring<XB> x;
            Ring<ST> y;
            for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of(p, i, x_tiles, x_rows);
                const Walk<KEYS> walk(p, it, y_rows);
                if (walk.count == 0) continue;
                const int buffer = x.at;
                fine = barrier_wait(&sm.x_free[buffer], x.parity ^ 1);
                if (!fine) break;
                barrier_expect(&sm.x_full[buffer], 2 * TERMS * x_rows * DP * 2);
#pragma unroll
                for (int k = 0; k < TERMS; ++k) {
                    load_rows<DP, kX>(sm.x[buffer][0][k], x0m, &sm.x_full[buffer], it.b + k * p.B, it.h, it.first);
                    load_rows<DP, kX>(sm.x[buffer][1][k], x1m, &sm.x_full[buffer], it.b + k * p.B, it.h, it.first);
                }
                ++done, x.next();
                for (int j = 0; fine && j < walk.count; ++j, ++n, y.next()) {
                    const int stage = y.at, row = (int)(walk[j] & 0x7fffffff) * y_rows;
                    fine = barrier_wait(&sm.y_free[stage], y.parity ^ 1);
                    if (!fine) break;
                    barrier_expect(&sm.y_full[stage], 2 * TERMS * y_rows * DP * 2);
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        load_rows<DP, kY>(sm.y[stage][0][k], y0m, &sm.y_full[stage], it.b + k * p.B, it.h, row);
                        load_rows<DP, kY>(sm.y[stage][1][k], y1m, &sm.y_full[stage], it.b + k * p.B, it.h, row);
                    }
                }
            }
            if (!fine) {     // nothing may still be on its way when the CTA ends
                for (int s = 0; s < XB; ++s)
                    if (done > s) barrier_wait(&sm.x_full[s], ((done - s + XB - 1) / XB - 1) & 1);
                for (int s = 0; s < ST; ++s)
                    if (n > s) barrier_wait(&sm.y_full[s], ((n - s + ST - 1) / ST - 1) & 1);
            }
        } else if (warp == kLast + 2 && KEYS) {
            // what the walked rows need beside their tiles
            Ring<ST> y;
            for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of(p, i, x_tiles, x_rows);
                const Walk<KEYS> walk(p, it, y_rows);
                for (int j = 0; fine && j < walk.count; ++j, y.next()) {
                    const int stage = y.at, tile = (int)walk[j];
                    float lse[2], delta[2];
                    uint4 see[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = lane + 32 * c, r = tile * y_rows + col;
                        const bool valid = col < y_rows && r < p.R;
                        lse[c] = valid ? (kScaled<T> ? kWeightExponent : 0.f) - p.lse[it.bh * p.R + r] : -INFINITY;
                        delta[c] = valid ? -p.delta[it.bh * p.R + r] : 0.f;
                        if (p.row_words != nullptr)
                            see[c] = valid ? __ldg(reinterpret_cast<const uint4 *>(row_words_of(p, it.b, it.h, r) + it.first / 32))
                                           : make_uint4(0, 0, 0, 0);
                    }
                    fine = barrier_wait(&sm.row_free[stage], y.parity ^ 1);
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
        } else if (warp == kLast + 1 && elect_one()) {
            constexpr uint32_t kScores = instruction(kBf16, kX, kY, false);
            constexpr uint32_t kGradients = instruction(kBf16, kX, DP, true);
            constexpr int kRow = kRowBytes<DP>;
            const uint32_t x0 = descriptor(smem_address(sm.x), 16), y0 = descriptor(smem_address(sm.y), 16),
                           z0 = descriptor(smem_address(sm.y), kY * 128);
            // Tiles whose products with P and dS are still to be issued, one fewer than there are groups: the scores
            // of a tile take the place of what the oldest one's products have read.
            struct Pending {
                int group;
                uint32_t turn;
                Ring<ST> y;
                Ring<AB> sums;
                bool first, last;
            } queue[kGroups - 1] = {};
            int waiting = 0;
            Ring<XB> x;
            Ring<ST> y;
            Ring<kGroups> groups;
            Ring<AB> sums;
            const auto issue_sums = [&] {
                const Pending t = queue[0];
#pragma unroll
                for (int i = 0; i + 1 < kGroups - 1; ++i) queue[i] = queue[i + 1];
                --waiting;
                const int group = t.group, stage = t.y.at;
                if (t.first) fine = fine && barrier_wait(&sm.acc_free[t.sums.at], t.sums.parity ^ 1);
                if (!KEYS && p.key_words != nullptr) fine = fine && barrier_wait(&sm.y_clean[stage], t.y.parity);
                fine = fine && barrier_wait(&sm.p_full[group], t.turn);
                fence_after();
                if (fine) {
                    const uint32_t from = tmem + group * kGroup, za = z0 + stage * (2 * TERMS * kYBytes >> 4);
                    const uint32_t acc = tmem + Sh::kAcc + t.sums.at * Sh::kSums;
#pragma unroll
                    for (int k = kPairs - kPairsOf; k < kPairs; ++k) {
                        const bool add = !t.first || k > kPairs - kPairsOf;
#pragma unroll
                        for (int j = 0; j < kY; j += 16) {
                            const uint32_t of = right_term(k) * kYBytes + j * kRow;
                            if constexpr (KEYS)
                                mma_ts<kRow>(acc, from + (left_term(k) == 2 ? Sh::third(true) : kS + 32 * left_term(k)) + j / 2, za + (TERMS * kYBytes + of >> 4), kGradients, add || j > 0);
                            mma_ts<kRow>(acc + (KEYS ? DP : 0), from + (left_term(k) == 2 ? Sh::third(false) : kT + 32 * left_term(k)) + j / 2, za + (of >> 4), kGradients, add || j > 0);
                        }
                    }
                    commit(&sm.y_free[stage]);
                    if (t.last) commit(&sm.acc_full[t.sums.at]);
                }
            };
            for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of(p, i, x_tiles, x_rows);
                const Walk<KEYS> walk(p, it, y_rows);
                if (walk.count == 0) continue;
                const int buffer = x.at;
                fine = barrier_wait(&sm.x_full[buffer], x.parity);
                for (int j = 0; fine && j < walk.count; ++j, y.next(), groups.next()) {
                    const int stage = y.at, group = groups.at;
                    fine = barrier_wait(&sm.y_full[stage], y.parity);
                    if (fine) {
                        const uint32_t to = tmem + group * kGroup;
                        const uint32_t xa = x0 + buffer * (2 * TERMS * kXBytes >> 4), ya = y0 + stage * (2 * TERMS * kYBytes >> 4);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int k = kPairs - kPairsOf; k < kPairs; ++k) {
#pragma unroll
                                for (int d = 0; d < DP; d += 16)
                                    mma<kRow>(to + (half == 0 ? kS : kT),
                                              xa + ((half * TERMS + left_term(k)) * kXBytes + (d & ~63) * kX * 2 + (d & 63) * 2 >> 4),
                                              ya + ((half * TERMS + right_term(k)) * kYBytes + (d & ~63) * kY * 2 + (d & 63) * 2 >> 4), kScores,
                                              d > 0 || k > kPairs - kPairsOf);
                            }
                        }
                        commit(&sm.s_full[group]);
                        if (j == walk.count - 1) commit(&sm.x_free[buffer]);
                    }
                    if (waiting == kGroups - 1) issue_sums();
                    const Pending t = {group, groups.parity, y, sums, j % Sh::kRun == 0, (j + 1) % Sh::kRun == 0 || j == walk.count - 1};
                    if (kGroups == 2 || waiting == 0) queue[0] = t; else queue[kGroups - 2] = t;
                    ++waiting;
                    if (t.last) sums.next();
                }
                x.next();
            }
            while (fine && waiting > 0) issue_sums();
        } else if (warp == kLast + 3 && !KEYS && p.key_words != nullptr) {
            // rows of k that nobody may see: their dS is 0 and its products have to be
            Ring<ST> y;
            for (unsigned i = blockIdx.x; fine && i < items; i += gridDim.x) {
                const Item it = item_of(p, i, x_tiles, x_rows);
                const Walk<KEYS> walk(p, it, y_rows);
                const uint32_t *words = key_words_of(p, it.b, it.h);
                for (int j = 0; fine && j < walk.count; ++j, y.next()) {
                    const uint32_t entry = walk[j];
                    const int stage = y.at;
                    // (whether their scores are formed before or after makes no difference: they are masked)
                    fine = barrier_wait(&sm.y_full[stage], y.parity);
                    if (fine && !(entry >> 31)) {
                        const uint2 see = __ldg(reinterpret_cast<const uint2 *>(words) + entry);
                        constexpr int kChunks = DP / 8;
                        for (int c = lane; c < 64 * kChunks; c += 32) {
                            const int r = c / kChunks;
                            if (!(((r < 32 ? see.x : see.y) >> (r & 31)) & 1)) {
#pragma unroll
                                for (int k = 0; k < TERMS; ++k)
                                    *reinterpret_cast<uint4 *>(sm.y[stage][0][k] + swizzled<DP, kY>(r, c % kChunks)) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        fence_async_shared();
                    }
                    barrier_arrive(&sm.y_clean[stage]);
                }
            }
        }
    }
    __syncthreads();
    if (warp == kLast) {
        __syncwarp();
        fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int DP, bool KEYS, int TERMS = 1>
cudaError_t launch(const AttentionParams &p, cudaStream_t stream) {
    const int row_tile = KEYS ? kY : kX, state_tile = KEYS ? kX : kY;
    tc::TensorMap q, g, k, v;
    if constexpr (TERMS == 3) {
        const int64_t D8 = (p.D + 7) / 8 * 8, heads = (int64_t)p.K * p.share;
        const int64_t rows[3] = {p.Q * heads * D8, heads * D8, D8}, states[3] = {(int64_t)p.S * p.K * D8, p.K * D8, D8};
        if (!tc::make_map<T, DP>(q, p.q_terms, rows, 3 * p.B, p.Q, p.K, p.share, (int)D8, row_tile) ||
            !tc::make_map<T, DP>(g, p.g_terms, rows, 3 * p.B, p.Q, p.K, p.share, (int)D8, row_tile) ||
            !tc::make_map<T, DP>(k, p.k_terms, states, 3 * p.B, p.S, p.K, 1, (int)D8, state_tile) ||
            !tc::make_map<T, DP>(v, p.v_terms, states, 3 * p.B, p.S, p.K, 1, (int)D8, state_tile))
            return cudaErrorNotSupported;
    } else {
        const int64_t gs[3] = {(int64_t)p.Q * p.K * p.share * p.D, (int64_t)p.K * p.share * p.D, p.D};
        if (!tc::make_map<T, DP>(q, p.q, p.qs, p.B, p.Q, p.K, p.share, p.D, row_tile) ||
            !tc::make_map<T, DP>(g, p.grad_out, gs, p.B, p.Q, p.K, p.share, p.D, row_tile) ||
            !tc::make_map<T, DP>(k, p.k, p.ks, p.B, p.S, p.K, 1, p.D, state_tile) ||
            !tc::make_map<T, DP>(v, p.v, p.vs, p.B, p.S, p.K, 1, p.D, state_tile))
            return cudaErrorNotSupported;
    }
    const auto kernel = attention_backward_tc_kernel<T, DP, KEYS, TERMS>;
    using Sh = Shape<DP, KEYS, TERMS>;
    static std::atomic<bool> fits{false};
    if (!fits) fits = tc::registers_suffice(kernel, Sh::kThreads, 128 * (Sh::kGroups * Sh::kRegisters + Sh::kFew + Sh::kWriting));
    if (!fits) return cudaErrorInvalidConfiguration;
    constexpr size_t smem = sizeof(Shared<DP, KEYS, TERMS>);
    static_assert(smem <= 227 * 1024);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int rows = row_tile / p.share * p.share;
    const int x_rows = KEYS ? kX : rows, y_rows = KEYS ? rows : kY;
    const int64_t items = (int64_t)p.B * p.K * p.splits * (((KEYS ? p.S : p.R) + x_rows - 1) / x_rows);
    if (items > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const unsigned grid = (unsigned)std::min<int64_t>(items, 148);
    return launch_dependent(kernel, dim3(grid), Shape<DP, KEYS, TERMS>::kThreads, smem, stream, p, KEYS ? k : q, KEYS ? v : g, KEYS ? q : k,
                            KEYS ? g : v, (unsigned)items, x_rows, y_rows);
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, bool keys, cudaStream_t stream) {
    if (p.D <= 32) return keys ? launch<T, 32, true>(p, stream) : launch<T, 32, false>(p, stream);
    if (p.D <= 64) return keys ? launch<T, 64, true>(p, stream) : launch<T, 64, false>(p, stream);
    return keys ? launch<T, 128, true>(p, stream) : launch<T, 128, false>(p, stream);
}

cudaError_t launch_float(const AttentionParams &p, bool keys, cudaStream_t stream) {
    using T = __nv_bfloat16;
    if (p.D <= 32) return keys ? launch<T, 32, true, 3>(p, stream) : launch<T, 32, false, 3>(p, stream);
    return keys ? launch<T, 64, true, 3>(p, stream) : launch<T, 64, false, 3>(p, stream);
}

}  // namespace

cudaError_t launch_attention_backward_tc(const AttentionParams &p, int dtype, bool keys, cudaStream_t stream) {
    return dtype == 0 ? launch_float(p, keys, stream)
           : dtype == 1 ? launch_typed<__half>(p, keys, stream) : launch_typed<__nv_bfloat16>(p, keys, stream);
}

}  // namespace msda_b200
