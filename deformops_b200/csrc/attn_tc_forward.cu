// Cross attention forward on the fifth-generation tensor cores, 16-bit types, and float32 up to 64 channels as three
// bf16 terms of every operand (TERMS = 3: six products for one).
//
// A CTA holds RT tiles of 128 rows and walks tiles of BN states.  One thread has TMA bring the tiles of
// k and v, one thread issues the products, and RT * KW groups of four warps do the softmax, a thread to
// a row: scores come from tensor memory, weights go back there (in the scores' place) as the left
// operand of the second product, whose sums stay in tensor memory until the end.
//
//   S = q k^T (BN columns)   P = exp2(c S - m) (BN / 2 columns, 16-bit)   O += P v (DP columns)
//
// KW groups share a row tile and take the state tiles in turn, each with a maximum, sum and O of its
// own; at the end the parts are weighted and added.  The work is bound by latencies of a group's cycle
// (scores, loads, exponentials, stores, product), so as many groups as tensor memory holds run at once:
// four with BN = 64 up to 64 channels, two with BN = 128 above.  Short passes are bound by the beginning and end of a
// CTA and take one group, 128 rows and a share of the SM: three CTAs to it, two above 64 channels (four of up to 64
// channels fit, with fewer registers: 19.0 us against 17.0 for 4 x 4096 rows of 8 heads over 64 states, and 30.7
// with big CTAs).
//
// The running maximum is only raised when a row would leave a range of 2^8 (float16: 2^4) above it: then the
// row's sums in tensor memory are scaled, which is rare after the first tiles, and exact in between (a
// weight of up to 2^8 rounds like one of 1).  float16 has no normal numbers below 2^-14: its weights are 2^7 times as large,
// and so is the sum that they are divided by (thousands of weights of 2^-21 beside one of 1 had 4 bits).  They are 2^11 at
// most, and 2^15 where scores are so large, 2^26, that a maximum is rounded by 2.
//
// 16-bit types: weights are rounded to the type, which a product's operands have to share.  Half a step each, independent of
// one another, is about what rounding the result costs once more: bf16 2.1e-3 off, a plain form rounded once 1.7e-3.
//
// 4 x 300 queries over 17 821 states, 8 heads of 32, bf16: 98 us (exponential unit and issue slots 48 %, tensor cores
// 14 %); 2 x 2048 over 4096, 16 heads on 4 of 128: 145 us a call among others, 950 TFLOP/s (160 alone, under a profiler).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace msda_b200 {

namespace {

constexpr int kTileRows = 128;

template <int DP, int RT, int KW, int TERMS>
struct Shape {
    static constexpr bool kSmall = RT * KW == 1;               // several CTAs to an SM
    static constexpr int BN = DP == 128 && !kSmall ? 128 : 64; // states of a tile
    // tiles of k and v in flight
    static constexpr int ST = kSmall ? 2 : DP == 128 || DP * TERMS > 128 ? KW + 1 : TERMS == 3 ? (RT == 1 ? 6 : 4) : 8;
    static constexpr int kGroups = RT * KW;
    static constexpr int kThreads = kGroups * 128 + 128;
    // columns of tensor memory of a group: S, in whose place P comes (a third term needs more), O
    static constexpr uint32_t kWeights = BN / 2, kO = std::max<uint32_t>(BN, TERMS * kWeights), kColumns = kO + DP;
    static constexpr int kAllocated = !kSmall ? 512 : kColumns <= 128 ? 128 : 256;
    static constexpr int kCtas = !kSmall ? 1 : std::min<int>(3, 512 / kAllocated);
    // what a thread may hold: all of the block's at launch, less what the last four warps need
    static constexpr int kRegisters = kSmall ? (kCtas == 3 ? 128 : 200) : kGroups == 4 ? 104 : 224;
    static constexpr int kFew = kSmall ? (kCtas == 3 ? 32 : 56) : kGroups == 4 ? 64 : 56;
    // Tiles after which a group takes its sums on in registers: those of the tensor cores are cut off, not rounded, at
    // every product that is added (2^-25.7 of the sum each, 24 times a tile with terms).  Four groups (up to 32 channels)
    // have no registers for it: those of two row tiles keep them in shared memory; those of one, which would have room for
    // five tiles in flight then and be 1.4 times slower, and small CTAs take few tiles instead.
    static constexpr bool kRuns = TERMS == 3 && (DP == 64 || RT == 2), kShared = kRuns && DP == 32;
    static constexpr int kRun = kRuns ? 4 : 1 << 30;
    static_assert(kGroups * kColumns <= 512);
    static_assert(ST > KW);                                    // a tile is freed KW tiles after its scores
};

template <int DP, int RT, int KW, int TERMS>
struct Shared {
    using Sh = Shape<DP, RT, KW, TERMS>;
    alignas(1024) unsigned char q[RT][TERMS][kTileRows * DP * 2];
    alignas(1024) unsigned char k[Sh::ST][TERMS][Sh::BN * DP * 2];
    alignas(1024) unsigned char v[Sh::ST][TERMS][Sh::BN * DP * 2];
    float m[Sh::kGroups][kTileRows], l[Sh::kGroups][kTileRows];
    float sums[Sh::kShared ? Sh::kGroups : 1][Sh::kShared ? DP : 1][kTileRows];      // of the runs so far
    uint64_t full[Sh::ST], clean[Sh::ST], free[Sh::ST];        // of a stage: its k and v
    uint64_t s_full[Sh::kGroups], p_full[Sh::kGroups], o_full[Sh::kGroups];
    uint32_t tmem;
};

// the BN / 32 mask words of a tile
template <int N>
struct Words {
    uint32_t w[N];
    __device__ __forceinline__ void load(const uint32_t *from, int tile) {
        if constexpr (N == 4) {
            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(from) + tile);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else {
            const uint2 x = __ldg(reinterpret_cast<const uint2 *>(from) + tile);
            w[0] = x.x, w[1] = x.y;
        }
    }
    __device__ __forceinline__ void existing(int S, int tile) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = key_word(nullptr, S, tile * N + i);
    }
    __device__ __forceinline__ bool all() const {
        uint32_t x = w[0];
#pragma unroll
        for (int i = 1; i < N; ++i) x &= w[i];
        return x == 0xffffffffu;
    }
};

template <typename T, int DP, int RT, int KW, int TERMS>
__global__ void __launch_bounds__(Shape<DP, RT, KW, TERMS>::kThreads, Shape<DP, RT, KW, TERMS>::kCtas)
    attention_forward_tc_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ tc::TensorMap km,
                                const __grid_constant__ tc::TensorMap vm) {
    using namespace tc;
    using Sh = Shape<DP, RT, KW, TERMS>;
    using Out = std::conditional_t<TERMS == 3, float, T>;      // of the call's tensors; T is that of the products
    constexpr int BN = Sh::BN, NW = BN / 32, ST = Sh::ST;
    constexpr uint32_t kO = Sh::kO, kP = Sh::kWeights;
    constexpr int kPairsOf = TERMS == 3 ? kPairs : 1, kTile = BN * DP * 2;
    constexpr int kLast = Sh::kGroups * 4;                     // first of the last four warps
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr float kUp = kScaled<T> ? 7.f : 0.f;              // exponent of what the weights are multiplied by
    constexpr float kAbove = kScaled<T> ? 4.f : 8.f;           // how far they may be above the maximum
    extern __shared__ __align__(1024) unsigned char raw[];
    auto &sm = *reinterpret_cast<Shared<DP, RT, KW, TERMS> *>(raw);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    const int row_tiles = (p.R + RT * kTileRows - 1) / (RT * kTileRows);
    const unsigned outer = blockIdx.x / row_tiles, of = outer / p.splits;
    const int first = (int)(blockIdx.x - outer * row_tiles) * RT * kTileRows, part = (int)(outer - of * p.splits);
    const int64_t bh = of;
    const int b = (int)(of / p.K), h = (int)(of - b * p.K);
    const uint32_t *words = key_words_of(p, b, h);

    if (warp == kLast + 1) tmem_alloc(&sm.tmem, Sh::kAllocated);
    if (warp == kLast && elect_one()) {
        for (int s = 0; s < ST; ++s) {
            barrier_init(&sm.full[s], 1), barrier_init(&sm.free[s], 1), barrier_init(&sm.clean[s], 32);
        }
        for (int g = 0; g < Sh::kGroups; ++g)
            barrier_init(&sm.s_full[g], 1), barrier_init(&sm.p_full[g], 128), barrier_init(&sm.o_full[g], 1);
        fence_async_shared();
    }
    __syncwarp();
    grid_dependency_wait();            // (of what this call has launched before: masks, terms)
    const Tiles<BN> tiles(p, b, h, part);
    const auto load = [&](int n, int stage) {
        const int state = (int)(tiles[n] & 0x7fffffff) * BN;
        barrier_expect(&sm.full[stage], 2 * TERMS * kTile);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
            load_rows<DP, BN>(sm.k[stage][i], km, &sm.full[stage], b + i * p.B, h, state);
            load_rows<DP, BN>(sm.v[stage][i], vm, &sm.full[stage], b + i * p.B, h, state);
        }
    };
    // the first tiles are on their way while the rows of q come
    if (warp == kLast && elect_one())
        for (int n = 0; n < ST && n < tiles.count; ++n) load(n, n);
    if (warp < 4 * RT) {
        // a thread to a row of q
        const int r = first + threadIdx.x;
        const Out *q = static_cast<const Out *>(p.q) + (r < p.R ? row_offset(p.qs, p.share, b, h, r) : 0);
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
            uint4 x[TERMS];
            if constexpr (TERMS == 3) {
                const uint4 none = make_uint4(0, 0, 0, 0);
                const uint4 f[2] = {r < p.R && c * 8 < p.D ? ldg16(q + c * 8) : none,
                                    r < p.R && c * 8 + 4 < p.D ? ldg16(q + c * 8 + 4) : none};
                uint32_t t[4][3];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    split_terms(make_float2(__uint_as_float(f[i].x), __uint_as_float(f[i].y)), t[2 * i]);
                    split_terms(make_float2(__uint_as_float(f[i].z), __uint_as_float(f[i].w)), t[2 * i + 1]);
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) x[i] = make_uint4(t[0][i], t[1][i], t[2][i], t[3][i]);
            } else {
                x[0] = r < p.R && c * 8 < p.D ? ldg16(q + c * 8) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < TERMS; ++i)
                *reinterpret_cast<uint4 *>(sm.q[warp >> 2][i] + swizzled<DP, kTileRows>(threadIdx.x & 127, c)) = x[i];
        }
        fence_async_shared();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    bool fine = true;

    if (warp < kLast) {
        registers_up<Sh::kRegisters>();
        const int group = warp >> 2, tile_of_rows = group % RT, way = group / RT, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t mine = tmem + group * Sh::kColumns + lanes;
        const int r = first + tile_of_rows * kTileRows + row;
        const bool idle = first + tile_of_rows * kTileRows + (row & ~31) >= p.R;       // a whole warp behind the last row
        const uint32_t *rw = r < p.R ? row_words_of(p, b, h, r) : nullptr;
        if (rw == nullptr) rw = words;
        float m = -INFINITY, l = 0.f;
        int done = 0;
        [[maybe_unused]] float sums[Sh::kRuns && !Sh::kShared ? DP : 1] = {};      // of the runs so far
        const auto take_on = [&](bool first_run) {
            if constexpr (Sh::kRuns) {
#pragma unroll
                for (int d = 0; d < DP; d += 16) {
                    uint32_t o[16];
                    tmem_load16(o, mine + kO + d);
                    tmem_wait_load();
                    loaded(o);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        if constexpr (Sh::kShared) {
                            float &sum = sm.sums[group][d + c][row];
                            sum = __uint_as_float(o[c]) + (first_run ? 0.f : sum);
                        } else {
                            sums[d + c] += __uint_as_float(o[c]);
                        }
                    }
                }
            }
        };
        const bool own_words = p.row_words != nullptr;
        uint32_t entry = way < tiles.count ? tiles[way] : 0;
        Words<NW> see{};
        if (rw != nullptr && way < tiles.count && (own_words || !(entry >> 31))) see.load(rw, entry & 0x7fffffff);
        for (int n = way; fine && n < tiles.count; n += KW, ++done) {
            // the next tile's mask comes while this one is worked on
            uint32_t entry_next = 0;
            Words<NW> see_next{};
            if (n + KW < tiles.count) {
                entry_next = tiles[n + KW];
                if (rw != nullptr && (own_words || !(entry_next >> 31))) see_next.load(rw, entry_next & 0x7fffffff);
            }
            fine = barrier_wait(&sm.s_full[group], done & 1);
            if (!fine) break;
            fence_after();
            if (!idle) {
                const bool starts = done % Sh::kRun == 0;          // a run; what was summed before lies there still
                if (starts && done > 0) take_on(done == Sh::kRun);
                uint32_t s[NW][32];
#pragma unroll
                for (int j = 0; j < NW; ++j) tmem_load32(s[j], mine + 32 * j);
                tmem_wait_load();
#pragma unroll
                for (int j = 0; j < NW; ++j) loaded(s[j]);
                if (own_words ? !__all_sync(0xffffffffu, see.all()) : !(entry >> 31)) {
                    if (rw == nullptr) see.existing(p.S, entry & 0x7fffffff);
#pragma unroll
                    for (int j = 0; j < NW; ++j)
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see.w[j] & (1u << c))) s[j][c] = 0xff800000u;        // -inf
                }
                float top[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    constexpr int kRun = BN / 4;
                    top[j] = __uint_as_float(s[j * kRun / 32][j * kRun % 32]);
#pragma unroll
                    for (int c = 1; c < kRun; ++c) top[j] = fmaxf(top[j], __uint_as_float(s[(j * kRun + c) / 32][(j * kRun + c) % 32]));
                }
                const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
                const bool raise = best > m + kAbove || (m == -INFINITY && best > m);
                if (__any_sync(0xffffffffu, raise)) {
                    const float to = raise ? best : m;
                    const float keep = to == -INFINITY ? 1.f : fast_exp2(m - to);
                    m = to;
                    l *= keep;
                    if constexpr (Sh::kShared) {
                        if (done >= Sh::kRun) {
#pragma unroll 8
                            for (int d = 0; d < DP; ++d) sm.sums[group][d][row] *= keep;
                        }
                    } else if constexpr (Sh::kRuns) {
#pragma unroll
                        for (int d = 0; d < DP; ++d) sums[d] *= keep;
                    }
                    if (!starts) {         // (that the scores are there says that the product before is done)
#pragma unroll
                        for (int d = 0; d < DP; d += 16) {
                            uint32_t o[16];
                            tmem_load16(o, mine + kO + d);
                            tmem_wait_load();
                            loaded(o);
#pragma unroll
                            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
                            tmem_store16(mine + kO + d, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m - kUp;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), less2 = make_float2(-base, -base);
                float2 sum[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    uint32_t w[TERMS][16];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float2 x = fma2(make_float2(__uint_as_float(s[j][c]), __uint_as_float(s[j][c + 1])), scale2, less2);
                        x.x = fast_exp2(x.x), x.y = fast_exp2(x.y);
                        sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], x);
                        if constexpr (TERMS == 3) {
                            uint32_t t[3];
                            split_terms(x, t);
                            w[0][c >> 1] = t[0], w[1][c >> 1] = t[1], w[TERMS - 1][c >> 1] = t[2];
                        } else {
                            w[0][c >> 1] = VecTraits<T>::pack2(x);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) tmem_store16(mine + i * kP + 16 * j, w[i]);
                }
                l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_store();
            }
            fence_before();
            barrier_arrive(&sm.p_full[group]);
            entry = entry_next;
            see = see_next;
        }
        // the groups of a row tile: every one adds a share of the columns of all
        if (done > 0) {
            fine = fine && barrier_wait(&sm.o_full[group], 0);
            fence_after();
        }
        if constexpr (Sh::kRuns) {
            if (done > Sh::kRun && !idle) {
                take_on(false);
#pragma unroll
                for (int d = 0; d < DP; d += 16) {
                    uint32_t o[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        if constexpr (Sh::kShared) o[c] = __float_as_uint(sm.sums[group][d + c][row]);
                        else o[c] = __float_as_uint(sums[d + c]);
                    }
                    tmem_store16(mine + kO + d, o);
                }
                tmem_wait_store();
            }
        }
        if (!fine) l = NAN;
        float factor[KW], lse;
        if constexpr (KW > 1) {
            sm.m[group][row] = m, sm.l[group][row] = l;
            fence_before();
            asm volatile("bar.sync 1, %0;" ::"n"(Sh::kGroups * 128) : "memory");
            fence_after();
            float best = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) best = fmaxf(best, sm.m[w * RT + tile_of_rows][row]);
            const float base = best == -INFINITY ? 0.f : best;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float lw = sm.l[w * RT + tile_of_rows][row];
                factor[w] = lw == 0.f ? 0.f : fast_exp2(sm.m[w * RT + tile_of_rows][row] - base);
                total += factor[w] * lw;
            }
#pragma unroll
            for (int w = 0; w < KW; ++w) factor[w] = total == 0.f ? 0.f : factor[w] / total;
            lse = total == 0.f ? (p.splits > 1 ? -INFINITY : INFINITY) : best - kUp + log2f(total);
        } else {
            factor[0] = l == 0.f ? 0.f : 1.f / l;
            lse = l == 0.f ? (p.splits > 1 ? -INFINITY : INFINITY) : m - kUp + log2f(l);
        }
        const int64_t at = bh * p.R + r, rows = (int64_t)p.B * p.K * p.R;
        const int query = r / p.share;
        Out *out = static_cast<Out *>(p.out) + (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (r - query * p.share)) * p.D;
        float *parts = p.part + (part * rows + at) * p.D;
        if (r < p.R && way == 0) (p.splits > 1 ? p.part_lse + part * rows : p.lse)[at] = lse;
        constexpr int kShare = DP / KW, kStep = kShare < 16 ? 8 : 16;
        if (!idle) {
#pragma unroll
            for (int d = 0; d < kShare; d += kStep) {
                const int col = way * kShare + d;
                float2 x[kStep / 2];
#pragma unroll
                for (int c = 0; c < kStep / 2; ++c) x[c] = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    uint32_t o[kStep];
                    const uint32_t from = tmem + (w * RT + tile_of_rows) * Sh::kColumns + lanes + kO + col;
                    if constexpr (kStep == 16) tmem_load16(o, from); else tmem_load8(o, from);
                    tmem_wait_load();
                    loaded(o);
                    // (a group that had no tile has never written its columns)
                    if (factor[w] != 0.f) {
#pragma unroll
                        for (int c = 0; c < kStep / 2; ++c)
                            ffma2(x[c], make_float2(__uint_as_float(o[2 * c]), __uint_as_float(o[2 * c + 1])), make_float2(factor[w], factor[w]));
                    }
                }
                if (r >= p.R) continue;
#pragma unroll
                for (int c = 0; c < kStep / 2; c += 4) {
                    if (col + 2 * c >= p.D) continue;
                    if (TERMS == 3 || p.splits > 1) {
                        float *to = p.splits > 1 ? parts : reinterpret_cast<float *>(out);
                        *reinterpret_cast<float4 *>(to + col + 2 * c) = make_float4(x[c].x, x[c].y, x[c + 1].x, x[c + 1].y);
                        if (col + 2 * c + 4 < p.D)
                            *reinterpret_cast<float4 *>(to + col + 2 * c + 4) = make_float4(x[c + 2].x, x[c + 2].y, x[c + 3].x, x[c + 3].y);
                    } else if constexpr (TERMS == 1) {
                        const float2 y[4] = {x[c], x[c + 1], x[c + 2], x[c + 3]};
                        *reinterpret_cast<uint4 *>(out + col + 2 * c) = VecTraits<T>::pack(y);
                    }
                }
            }
        }
        fence_before();
    } else {
        registers_down<Sh::kFew>();
        if (warp == kLast && elect_one()) {
            int n = min(ST, tiles.count);
            Ring<ST> ring;
            ring.next(n);
            for (; fine && n < tiles.count; ++n, ring.next()) {
                fine = barrier_wait(&sm.free[ring.at], ring.parity ^ 1);
                if (!fine) break;
                load(n, ring.at);
            }
            // nothing may still be on its way when the CTA ends
            for (int s = 0; s < ST && !fine; ++s) {
                const int turns = (n - s + ST - 1) / ST;
                if (turns > 0) barrier_wait(&sm.full[s], (turns - 1) & 1);
            }
        } else if (warp == kLast + 1 && elect_one()) {
            constexpr uint32_t kScores = instruction(kBf16, kTileRows, BN, false);
            constexpr uint32_t kOut = instruction(kBf16, kTileRows, DP, true);
            constexpr int kRow = kRowBytes<DP>;
            // The n-th tile is the groups' n % KW and their n / KW-th.  Its scores take the place of the weights of
            // their tile before, so the product with those is issued first: products are done in order.
            const uint32_t q0 = descriptor(smem_address(sm.q), 16), k0 = descriptor(smem_address(sm.k), 16),
                           v0 = descriptor(smem_address(sm.v), BN * 128);
            int n = 0;
            Ring<ST> now, then;                // of tiles n and n - KW
            for (int round = 0; fine && n < tiles.count + KW; ++round) {
#pragma unroll
                for (int w = 0; w < KW; ++w, ++n) {
                    const bool scores = n < tiles.count, weights = round > 0 && n - KW < tiles.count;
                    const int stage = now.at, last = then.at;
                    if (scores) fine = fine && barrier_wait(&sm.full[stage], now.parity);
                    if (weights && words != nullptr) fine = fine && barrier_wait(&sm.clean[last], then.parity);
                    now.next();
                    if (round > 0) then.next();
                    const uint32_t ka = k0 + stage * (TERMS * kTile >> 4), va = v0 + last * (TERMS * kTile >> 4);
#pragma unroll
                    for (int q = 0; q < RT; ++q) {
                        const int group = w * RT + q;
                        const uint32_t at = tmem + group * Sh::kColumns;
                        if (weights) {
                            fine = fine && barrier_wait(&sm.p_full[group], (round - 1) & 1);
                            if (!fine) break;
                            fence_after();
#pragma unroll
                            for (int i = kPairs - kPairsOf; i < kPairs; ++i) {
#pragma unroll
                                for (int j = 0; j < BN; j += 16)
                                    mma_ts<kRow>(at + kO, at + left_term(i) * kP + j / 2, va + (right_term(i) * kTile + j * kRow >> 4), kOut,
                                                 (round - 1) % Sh::kRun != 0 || j > 0 || i > kPairs - kPairsOf);
                            }
                            if (q == RT - 1) commit(&sm.free[last]);
                            if (!scores) commit(&sm.o_full[group]);
                        }
                        if (scores && fine) {
#pragma unroll
                            for (int i = kPairs - kPairsOf; i < kPairs; ++i) {
#pragma unroll
                                for (int d = 0; d < DP; d += 16)
                                    mma<kRow>(at, q0 + (((q * TERMS + left_term(i)) * DP + (d & ~63)) * kTileRows * 2 + (d & 63) * 2 >> 4),
                                              ka + (right_term(i) * kTile + (d & ~63) * BN * 2 + (d & 63) * 2 >> 4), kScores,
                                              d > 0 || i > kPairs - kPairsOf);
                            }
                            commit(&sm.s_full[group]);
                        }
                    }
                }
            }
        } else if (warp == kLast + 2 && words != nullptr) {
            // rows of v that nobody may see: whatever they hold, their weight is 0 and has to stay it
            Ring<ST> ring;
            for (int n = 0; fine && n < tiles.count; ++n, ring.next()) {
                const uint32_t entry = tiles[n];
                const int stage = ring.at;
                fine = barrier_wait(&sm.full[stage], ring.parity);
                if (fine && !(entry >> 31)) {
                    Words<NW> see;
                    see.load(words, entry);
                    constexpr int kChunks = DP / 8;
#pragma unroll
                    for (int j = 0; j < NW; ++j)
                        for (int c = lane; c < 32 * kChunks; c += 32)
                            if (!((see.w[j] >> (c / kChunks)) & 1)) {
#pragma unroll
                                for (int i = 0; i < TERMS; ++i)
                                    *reinterpret_cast<uint4 *>(sm.v[stage][i] + swizzled<DP, BN>(32 * j + c / kChunks, c % kChunks)) =
                                        make_uint4(0, 0, 0, 0);
                            }
                    fence_async_shared();
                }
                barrier_arrive(&sm.clean[stage]);
            }
        }
    }
    __syncthreads();
    if (warp == kLast + 1) {
        __syncwarp();
        fence_after();
        tmem_free(tmem, Sh::kAllocated);
    }
}

template <typename T, int DP, int RT, int KW, int TERMS = 1>
cudaError_t launch(const AttentionParams &p, cudaStream_t stream) {
    using Sh = Shape<DP, RT, KW, TERMS>;
    tc::TensorMap km, vm;
    if constexpr (TERMS == 3) {
        const int64_t D8 = (p.D + 7) / 8 * 8, dense[3] = {(int64_t)p.S * p.K * D8, p.K * D8, D8};
        if (!tc::make_map<T, DP>(km, p.k_terms, dense, 3 * p.B, p.S, p.K, 1, (int)D8, Sh::BN) ||
            !tc::make_map<T, DP>(vm, p.v_terms, dense, 3 * p.B, p.S, p.K, 1, (int)D8, Sh::BN))
            return cudaErrorNotSupported;
        TermsParams terms = {{{p.k, p.k_terms, {p.ks[0], p.ks[1], p.ks[2]}, p.S, p.K}, {p.v, p.v_terms, {p.vs[0], p.vs[1], p.vs[2]}, p.S, p.K}},
                             2, p.B, p.D};
        const cudaError_t e = launch_attention_terms(terms, stream);
        if (e != cudaSuccess) return e;
    } else if (!tc::make_map<T, DP>(km, p.k, p.ks, p.B, p.S, p.K, 1, p.D, Sh::BN) ||
               !tc::make_map<T, DP>(vm, p.v, p.vs, p.B, p.S, p.K, 1, p.D, Sh::BN)) {
        return cudaErrorNotSupported;
    }
    const auto kernel = attention_forward_tc_kernel<T, DP, RT, KW, TERMS>;
    static std::atomic<bool> fits{false};
    if (!fits) fits = tc::registers_suffice(kernel, Sh::kThreads, 128 * (Sh::kGroups * Sh::kRegisters + Sh::kFew));
    if (!fits) return cudaErrorInvalidConfiguration;
    constexpr size_t smem = sizeof(Shared<DP, RT, KW, TERMS>);
    static_assert((smem + 1024) * Sh::kCtas <= 228 * 1024);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)p.B * p.K * p.splits * ((p.R + RT * kTileRows - 1) / (RT * kTileRows));
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, dim3((unsigned)grid), Sh::kThreads, smem, stream, p, km, vm);
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, int row_tiles, cudaStream_t stream) {
    if (row_tiles == 0) return p.D <= 32 ? launch<T, 32, 1, 1>(p, stream) : p.D <= 64 ? launch<T, 64, 1, 1>(p, stream) : launch<T, 128, 1, 1>(p, stream);
    if (p.D <= 32) return row_tiles == 1 ? launch<T, 32, 1, 4>(p, stream) : launch<T, 32, 2, 2>(p, stream);
    if (p.D <= 64) return row_tiles == 1 ? launch<T, 64, 1, 4>(p, stream) : launch<T, 64, 2, 2>(p, stream);
    return row_tiles == 1 ? launch<T, 128, 1, 2>(p, stream) : launch<T, 128, 2, 1>(p, stream);
}

cudaError_t launch_float(const AttentionParams &p, int row_tiles, cudaStream_t stream) {
    using T = __nv_bfloat16;
    if (row_tiles == 0) return launch<T, 32, 1, 1, 3>(p, stream);
    if (p.D <= 32) return row_tiles == 1 ? launch<T, 32, 1, 4, 3>(p, stream) : launch<T, 32, 2, 2, 3>(p, stream);
    return row_tiles == 1 ? launch<T, 64, 1, 2, 3>(p, stream) : launch<T, 64, 2, 1, 3>(p, stream);
}

}  // namespace

cudaError_t launch_attention_forward_tc(const AttentionParams &p, int dtype, int row_tiles, cudaStream_t stream) {
    return dtype == 0 ? launch_float(p, row_tiles, stream)
           : dtype == 1 ? launch_typed<__half>(p, row_tiles, stream) : launch_typed<__nv_bfloat16>(p, row_tiles, stream);
}

}  // namespace msda_b200
