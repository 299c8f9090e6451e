// Cross attention of float32 with 65 to 128 channels on the fifth-generation tensor cores, forward and backward: three
// bf16 terms of every operand, six products for one.
//
// A CTA holds 128 rows of one side as the left operand and walks tiles of 64 of the other:
//
//              held X     walked Y, Z     w of a tile                         sums
//   FORWARD    q          k, v            P = exp2(c q k^T - max)             o  += P v
//   VALUES     k          q, do           P = exp2(c k q^T - L)               dv += P do
//   KEYS       k, v       q, do           dS = P (v do^T - delta)             dk += dS q
//   ROWS       q, do      k, v            dS = P (do v^T - delta)             dq += dS k
//
// Terms of 128 channels fill the memories: 128 rows take 192 columns of tensor memory or 96 KB of shared memory, a
// walked tile 48 KB.  So X's terms stay in tensor memory, which also spares the products a reading of 4 KB each (32
// cycles a product of N = 64 in place of 48), dv and dk are passes of their own (eight products in place of seven),
// and the second held operand has its first term, which half of the products use, in tensor memory and the others in
// shared memory:
//
//   columns    0 .. 191 X    192 .. 319 sums    320 .. 511: scores of two tiles, in whose places their weights' terms
//              come (FORWARD, VALUES); or scores, in whose place dS comes, and the second operand's first term
//
// FORWARD and VALUES have the scores of the next tile formed while one warpgroup, a thread to a row, works on this
// one's: bound by the tensor cores, 96 products of 32 cycles a tile.  KEYS and ROWS have no columns left for that; two
// warpgroups share the columns of a tile, and the tensor cores wait for them.  2 x 2048 queries over 4096 states, 16
// heads on 4 of 128 channels: 573 us forward and 2642 us backward (1440 and 1250 TFLOP/s of bf16 products); products of
// tf32 terms by warps took 20 ms for both.
#include <atomic>

#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace msda_b200 {

namespace {

enum Mode { FORWARD, VALUES, KEYS, ROWS };

constexpr int kX = 128, kY = 64, kD = 128, kTile = kY * kD * 2;        // (bytes of a term of a walked tile)
// Tiles after which the sums are taken on in registers: those of the tensor cores are cut off, not rounded, at every
// product that is added (2^-25.7 of the sum each, 24 times a tile).  Normal inputs over 2048 states: 1.4e-5 off without,
// 3.3e-6 with runs of eight tiles, 1.6e-6 with four; a run costs a reading of the sums, 1 % of its time.
constexpr int kRun = 4;
constexpr uint32_t kSums = 192, kScores = 320, kBuffer = 96, kSecond = 448;

template <Mode M>
struct Shape {
    static constexpr bool kOne = M == FORWARD || M == VALUES;          // one product of scores, two tiles under way
    static constexpr bool kHoldsRows = M == FORWARD || M == ROWS;
    static constexpr int kGroups = kOne ? 1 : 2, kThreads = 128 * kGroups + 256, kZ = kOne ? 2 : 1;
    // what a thread may hold: all of the block's at launch, shared out anew
    static constexpr int kRegisters = kOne ? 200 : 144, kSumming = kOne ? 200 : 144, kFew = kOne ? 104 : 80;
};

template <Mode M>
struct Shared {
    alignas(1024) unsigned char y[2][3][kTile];
    alignas(1024) unsigned char z[Shape<M>::kZ][3][kTile];
    alignas(1024) unsigned char x[Shape<M>::kOne ? 1 : 2][Shape<M>::kOne ? 16 : kX * kD * 2];      // second and third term of X1
    float m[2][kX], l[kX];              // FORWARD: the maximum that a run's sums go by; the sum of all weights
    uint64_t y_full[2], y_free[2], z_full[2], z_free[2], clean[2], s_full[2], p_full[2], done, run_full, run_free, m_full[2], l_full, drained;
    uint32_t tmem;
};

template <Mode M>
__global__ void __launch_bounds__(Shape<M>::kThreads, 1)
    attention_wide_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ tc::TensorMap ym,
                          const __grid_constant__ tc::TensorMap zm, int y_rows) {
    using namespace tc;
    using Sh = Shape<M>;
    constexpr bool kOne = Sh::kOne, kHoldsRows = Sh::kHoldsRows;
    constexpr int kGroups = Sh::kGroups, kZ = Sh::kZ, kLast = 4 * kGroups;
    extern __shared__ __align__(1024) unsigned char raw[];
    auto &sm = *reinterpret_cast<Shared<M> *>(raw);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    const int held = kHoldsRows ? p.R : p.S, x_tiles = (held + kX - 1) / kX;
    const unsigned outer = blockIdx.x / x_tiles, bh = outer / p.splits;
    const int first = (int)(blockIdx.x - outer * x_tiles) * kX, part = (int)(outer - bh * p.splits);
    const int b = (int)(bh / p.K), h = (int)(bh - b * p.K);
    const uint32_t *words = key_words_of(p, b, h);

    if (warp == kLast) tmem_alloc(&sm.tmem, 512);
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            barrier_init(&sm.y_full[s], 1), barrier_init(&sm.y_free[s], 1), barrier_init(&sm.z_full[s], 1), barrier_init(&sm.z_free[s], 1);
            barrier_init(&sm.clean[s], 32), barrier_init(&sm.s_full[s], 1), barrier_init(&sm.p_full[s], 128 * kGroups);
        }
        barrier_init(&sm.done, 1), barrier_init(&sm.run_full, 1), barrier_init(&sm.run_free, 128);
        barrier_init(&sm.m_full[0], 128), barrier_init(&sm.m_full[1], 128), barrier_init(&sm.l_full, 128), barrier_init(&sm.drained, 1);
        fence_async_shared();
    }
    if (y_rows < kY) {      // rows that no load reaches
        constexpr int kY16 = sizeof(sm.y) / 16, kZ16 = sizeof(sm.z) / 16;
        for (int i = threadIdx.x; i < kY16 + kZ16; i += Sh::kThreads)
            (i < kY16 ? reinterpret_cast<uint4 *>(sm.y)[i] : reinterpret_cast<uint4 *>(sm.z)[i - kY16]) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
    }
    grid_dependency_wait();            // (of what this call has launched before: masks, terms, delta)
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);

    // the tiles walked: listed ones of states, or all of the rows where anybody sees the held states
    const Tiles<kY> listed(p, b, h, part);
    int begin = 0, count = listed.count;
    if constexpr (!kHoldsRows) {
        Tiles<kY>::stretch((p.R + y_rows - 1) / y_rows, p.splits, part, begin, count);
        if (words != nullptr) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(words + first / 32));
            if ((w.x | w.y | w.z | w.w) == 0) count = 0;
        }
    }
    const auto tile_at = [&](int n) { return kHoldsRows ? listed[n] : (uint32_t)(begin + n); };

    const int group = warp >> 2, row = threadIdx.x & 127, x = first + row;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
    if (warp < kLast) {
        // a thread to a row of what is held
        const int64_t dense[3] = {(int64_t)p.Q * p.K * p.share * p.D, (int64_t)p.K * p.share * p.D, p.D};
        const float *from;
        if constexpr (kHoldsRows)
            from = static_cast<const float *>(group == 0 ? p.q : p.grad_out) +
                   (x < held ? (group == 0 ? row_offset(p.qs, p.share, b, h, x) : row_offset(dense, p.share, b, h, x)) : 0);
        else
            from = static_cast<const float *>(group == 0 ? p.k : p.v) +
                   (x < held ? (group == 0 ? b * p.ks[0] + x * p.ks[1] + h * p.ks[2] : b * p.vs[0] + x * p.vs[1] + h * p.vs[2]) : 0);
#pragma unroll
        for (int d = 0; d < kD; d += 32) {
            uint32_t t[3][16];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const uint4 f = x < held && d + 4 * c < p.D ? ldg16(from + d + 4 * c) : make_uint4(0, 0, 0, 0);
                uint32_t u[2][3];
                split_terms(make_float2(__uint_as_float(f.x), __uint_as_float(f.y)), u[0]);
                split_terms(make_float2(__uint_as_float(f.z), __uint_as_float(f.w)), u[1]);
#pragma unroll
                for (int i = 0; i < 3; ++i) t[i][2 * c] = u[0][i], t[i][2 * c + 1] = u[1][i];
            }
            if (group == 0) {
#pragma unroll
                for (int i = 0; i < 3; ++i) tmem_store16(mine + 64 * i + d / 2, t[i]);
            } else {
                tmem_store16(mine + kSecond + d / 2, t[0]);
                if constexpr (!kOne) {
#pragma unroll
                    for (int i = 1; i < 3; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<uint4 *>(sm.x[i - 1] + swizzled<kD, kX>(row, d / 8 + c)) =
                                make_uint4(t[i][4 * c], t[i][4 * c + 1], t[i][4 * c + 2], t[i][4 * c + 3]);
                }
            }
        }
        tmem_wait_store();
        if constexpr (!kOne) fence_async_shared();
    }
    fence_before();
    __syncthreads();
    fence_after();
    bool fine = true;

    if (warp < kLast) {
        registers_up<Sh::kRegisters>();
        const bool valid = x < held, idle = first + (row & ~31) >= held;       // (a whole warp behind the last row)
        const bool own_words = p.row_words != nullptr;
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
        constexpr int NW = kOne ? 2 : 1;                                       // words of 32 columns that a thread has
        const int w0 = kOne ? 0 : group;
        const uint32_t *rw = kHoldsRows && valid ? row_words_of(p, b, h, x) : nullptr;
        if (rw == nullptr) rw = words;
        const bool seen = valid && (kHoldsRows || ((key_word(words, p.S, x >> 5) >> (x & 31)) & 1));
        float my_lse = -INFINITY, my_delta = 0.f;                              // ROWS: both with the sign turned
        if (M == ROWS && valid) my_lse = -p.lse[(int64_t)bh * p.R + x], my_delta = -p.delta[(int64_t)bh * p.R + x];
        float m = -INFINITY, l = 0.f;                                          // FORWARD: running maximum and sum
        for (int n = 0; fine && n < count; ++n) {
            const uint32_t entry = tile_at(n);
            const int tile = (int)(entry & 0x7fffffff);
            const bool whole = entry >> 31;                                    // (of states)
            // which columns this row may use; `some`: not all, for some row of the warp
            uint32_t see[NW];
            bool some;
            float lse[NW], delta[NW];                                          // of column `lane` of a word: KEYS, VALUES
            if constexpr (kHoldsRows) {
#pragma unroll
                for (int j = 0; j < NW; ++j)
                    see[j] = rw == nullptr ? key_word(nullptr, p.S, 2 * tile + w0 + j)
                             : own_words || !whole ? __ldg(rw + 2 * tile + w0 + j) : 0xffffffffu;
                some = own_words ? !__all_sync(0xffffffffu, (see[0] & see[NW - 1]) == 0xffffffffu) : !whole;
            } else {
                some = own_words || !__all_sync(0xffffffffu, seen);
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    const int col = 32 * (w0 + j) + lane, r = tile * y_rows + col;
                    const bool there = col < y_rows && r < p.R;
                    lse[j] = there ? -p.lse[(int64_t)bh * p.R + r] : -INFINITY;
                    delta[j] = M == KEYS && there ? -p.delta[(int64_t)bh * p.R + r] : 0.f;
                    see[j] = seen ? 0xffffffffu : 0u;
                    if (own_words) {      // from a word to a column to a word to a row
                        const uint32_t word = there && !idle ? __ldg(row_words_of(p, b, h, r) + first / 32 + (warp & 3)) : 0u;
                        uint32_t turned = 0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const uint32_t of = __ballot_sync(0xffffffffu, (word >> i) & 1);
                            if (lane == i) turned = of;
                        }
                        see[j] &= turned;
                    }
                }
            }
            const int buffer = n & 1;
            fine = barrier_wait(&sm.s_full[buffer], (n >> 1) & 1);
            if (kOne && !fine) break;
            fence_after();
            const uint32_t at = mine + kScores + (kOne ? buffer * kBuffer : 0);
            uint32_t s[NW][32], t[kOne ? 1 : 32];
            if (!idle) {
#pragma unroll
                for (int j = 0; j < NW; ++j) tmem_load32(s[j], at + 32 * (w0 + j));
                if constexpr (!kOne) tmem_load32(t, at + 64 + 32 * group);
                tmem_wait_load();
#pragma unroll
                for (int j = 0; j < NW; ++j) loaded(s[j]);
                if constexpr (!kOne) loaded(t);
            }
            if constexpr (!kOne) {      // what either group stores takes the place of what the other loads
                fence_before();
                uint32_t all_fine;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                             : "=r"(all_fine)
                             : "r"((uint32_t)fine), "n"(kGroups * 128)
                             : "memory");
                fence_after();
                fine = all_fine != 0;
                if (!fine) break;
            }
            if (!idle) {
                float2 less2 = make_float2(my_lse, my_lse), sum[2];
                if constexpr (M == FORWARD) {
                    if (some) {
#pragma unroll
                        for (int j = 0; j < NW; ++j)
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!(see[j] & (1u << c))) s[j][c] = 0xff800000u;        // -inf
                    }
                    float top[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        top[j] = __uint_as_float(s[j / 2][j % 2 * 16]);
#pragma unroll
                        for (int c = 1; c < 16; ++c) top[j] = fmaxf(top[j], __uint_as_float(s[j / 2][j % 2 * 16 + c]));
                    }
                    const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
                    // the maximum is raised where a weight would leave exp2's range of 2^8 above it
                    const bool raise = best > m + 8.f || (m == -INFINITY && best > m);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float to = raise ? best : m;
                        const float keep = to == -INFINITY ? 1.f : fast_exp2(m - to);
                        m = to;
                        l *= keep;
                        if (n % kRun != 0) {       // (else the sums begin anew)
                            fine = barrier_wait(&sm.done, (n - 1) & 1);
                            fence_after();
#pragma unroll
                            for (int d = 0; d < kD; d += 16) {
                                uint32_t o[16];
                                tmem_load16(o, mine + kSums + d);
                                tmem_wait_load();
                                loaded(o);
#pragma unroll
                                for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
                                tmem_store16(mine + kSums + d, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    less2 = make_float2(-base, -base);
                    sum[0] = make_float2(l, 0.f), sum[1] = make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    uint32_t w[3][16];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        if constexpr (!kHoldsRows)
                            less2 = make_float2(__shfl_sync(0xffffffffu, lse[j], c), __shfl_sync(0xffffffffu, lse[j], c + 1));
                        float2 e = fma2(make_float2(__uint_as_float(s[j][c]), __uint_as_float(s[j][c + 1])), scale2, less2);
                        e.x = fast_exp2(e.x), e.y = fast_exp2(e.y);
                        if constexpr (M == FORWARD) sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], e);
                        if constexpr (!kOne) {
                            float2 d2 = make_float2(my_delta, my_delta);
                            if constexpr (M == KEYS)
                                d2 = make_float2(__shfl_sync(0xffffffffu, delta[j], c), __shfl_sync(0xffffffffu, delta[j], c + 1));
                            e = fmul2(e, add2(make_float2(__uint_as_float(t[c]), __uint_as_float(t[c + 1])), d2));
                        }
                        if (M != FORWARD && some) {      // (whatever an unseen state holds)
                            if (!((see[j] >> c) & 1)) e.x = 0.f;
                            if (!((see[j] >> c) & 2)) e.y = 0.f;
                        }
                        uint32_t u[3];
                        split_terms(e, u);
                        w[0][c >> 1] = u[0], w[1][c >> 1] = u[1], w[2][c >> 1] = u[2];
                    }
#pragma unroll
                    for (int i = 0; i < 3; ++i) tmem_store16(at + 32 * i + 16 * (w0 + j), w[i]);
                }
                if constexpr (M == FORWARD) l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_store();
            }
            if (kOne && n > 0) fine = barrier_wait(&sm.done, (n - 1) & 1) && fine;       // (every phase is waited for)
            if (M == FORWARD && (n % kRun == kRun - 1 || n == count - 1)) {
                const int run = n / kRun & 1;      // (what it held two runs before is read: the run before has begun)
                sm.m[run][row] = m;
                barrier_arrive(&sm.m_full[run]);
            }
            fence_before();
            barrier_arrive(&sm.p_full[buffer]);
        }
        if constexpr (M == FORWARD) {
            if (!fine) l = NAN;
            const float lse = l == 0.f ? (p.splits > 1 ? -INFINITY : INFINITY) : m + log2f(l);
            if (valid) (p.splits > 1 ? p.part_lse + part * ((int64_t)p.B * p.K * held) : p.lse)[(int64_t)bh * held + x] = lse;
            sm.l[row] = l;
            barrier_arrive(&sm.l_full);
        }
    } else if (warp >= kLast + 4) {
        // the sums, a thread to a row
        registers_up<Sh::kSumming>();
        const bool valid = x < held, idle = first + (row & ~31) >= held;
        float sum[kD], m = -INFINITY;
#pragma unroll
        for (int d = 0; d < kD; ++d) sum[d] = 0.f;
        for (int n = 0, run = 0; fine && n < count; n += kRun, ++run) {
            float keep = 1.f;
            if constexpr (M == FORWARD) {
                fine = barrier_wait(&sm.m_full[run & 1], (run >> 1) & 1);
                const float to = sm.m[run & 1][row];
                keep = to == -INFINITY ? 1.f : fast_exp2(m - to);
                m = to;
            }
            fine = barrier_wait(&sm.run_full, run & 1) && fine;
            if (!fine) break;
            fence_after();
            if (!idle) {
#pragma unroll
                for (int d = 0; d < kD; d += 16) {
                    uint32_t o[16];
                    tmem_load16(o, mine + kSums + d);
                    tmem_wait_load();
                    loaded(o);
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        sum[d + c] = M == FORWARD ? fmaf(sum[d + c], keep, __uint_as_float(o[c])) : sum[d + c] + __uint_as_float(o[c]);
                }
            }
            fence_before();
            barrier_arrive(&sm.run_free);
        }
        float factor = M == VALUES ? 1.f : p.scale;
        if constexpr (M == FORWARD) {
            fine = barrier_wait(&sm.l_full, 0) && fine;
            const float l = sm.l[row];
            factor = l == 0.f ? 0.f : 1.f / l;
        }
        if (!fine) factor = NAN;
        float *to = static_cast<float *>(M == FORWARD ? p.out : M == VALUES ? p.dv : M == KEYS ? p.dk : p.dq);
        if (p.splits > 1) {
            to = (M == VALUES ? p.part2 : p.part) + (part * ((int64_t)p.B * p.K * held) + (int64_t)bh * held + x) * p.D;
        } else if constexpr (kHoldsRows) {
            const int query = x / p.share;
            to += (((int64_t)b * p.Q + query) * p.K * p.share + h * p.share + (x - query * p.share)) * p.D;
        } else {
            to += (((int64_t)b * p.S + x) * p.K + h) * p.D;
        }
        if (valid) {
#pragma unroll
            for (int d = 0; d < kD; d += 4) {
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (factor != 0.f) f = make_float4(sum[d] * factor, sum[d + 1] * factor, sum[d + 2] * factor, sum[d + 3] * factor);
                if (d < p.D) *reinterpret_cast<float4 *>(to + d) = f;
            }
        }
    } else {
        registers_down<Sh::kFew>();
        if (warp == kLast && elect_one()) {
            // loads, in the order in which their places get free: Y is one tile ahead
            int ny = 0, nz = 0;
            const auto load = [&](bool second, int &n) {
                const bool two = !second || kZ == 2;
                const int stage = two ? n & 1 : 0;
                const uint32_t turn = two ? (n >> 1) & 1 : n & 1;
                fine = fine && barrier_wait(second ? &sm.z_free[stage] : &sm.y_free[stage], turn ^ 1);
                if (!fine) return;
                uint64_t *full = second ? &sm.z_full[stage] : &sm.y_full[stage];
                const int at = (int)(tile_at(n) & 0x7fffffff) * y_rows;
                barrier_expect(full, 3 * y_rows * kD * 2);
                for (int i = 0; i < 3; ++i)
                    load_rows<kD, kY>(second ? sm.z[stage][i] : sm.y[stage][i], second ? zm : ym, full, b + i * p.B, h, at);
                ++n;
            };
            if (count > 0) load(false, ny);
            while (fine && nz < count) {
                if (kOne && ny < count) load(false, ny);
                if (fine) load(true, nz);
                if (!kOne && fine && ny < count) load(false, ny);
            }
            if (!fine) {     // nothing may still be on its way when the CTA ends
                for (int s = 0; s < 2; ++s)
                    if (ny > s) barrier_wait(&sm.y_full[s], ((ny - s + 1) / 2 - 1) & 1);
                for (int s = 0; s < kZ; ++s)
                    if (nz > s) barrier_wait(&sm.z_full[s], ((nz - s + kZ - 1) / kZ - 1) & 1);
            }
        } else if (warp == kLast + 1 && elect_one()) {
            constexpr uint32_t kOf = instruction(true, kX, kY, false), kAdd = instruction(true, kX, kD, true);
            constexpr int kTerm = kTile >> 4, kHeld = kX * kD * 2 >> 4;
            const uint32_t y0 = descriptor(smem_address(sm.y), 16), z0 = descriptor(smem_address(sm.z), 16), x0 = descriptor(smem_address(sm.x), 16);
            const uint32_t sums_of = descriptor(kOne ? smem_address(sm.z) : smem_address(sm.y), kY * 128);
            const auto scores = [&](int n) {
                fine = fine && barrier_wait(&sm.y_full[n & 1], (n >> 1) & 1);
                if (!fine) return;
                const uint32_t to = tmem + kScores + (kOne ? (n & 1) * kBuffer : 0), ya = y0 + (n & 1) * 3 * kTerm;
    #pragma unroll
                for (int i = 0; i < kPairs; ++i)
    #pragma unroll
                    for (int d = 0; d < kD; d += 16)
                        mma_ts<128>(to, tmem + 64 * left_term(i) + d / 2, ya + right_term(i) * kTerm + ((d & 64) * kY * 2 + (d & 63) * 2 >> 4), kOf,
                                    i > 0 || d > 0);
                if constexpr (kOne) {
                    commit(&sm.y_free[n & 1]);
                } else {
                    fine = barrier_wait(&sm.z_full[0], n & 1);
                    if (!fine) return;
    #pragma unroll
                    for (int i = 0; i < kPairs; ++i)
    #pragma unroll
                        for (int d = 0; d < kD; d += 16) {
                            const uint32_t za = z0 + right_term(i) * kTerm + ((d & 64) * kY * 2 + (d & 63) * 2 >> 4);
                            if (left_term(i) == 0)
                                mma_ts<128>(to + 64, tmem + kSecond + d / 2, za, kOf, i > 0 || d > 0);
                            else
                                mma<128>(to + 64, x0 + (left_term(i) - 1) * kHeld + ((d & 64) * kX * 2 + (d & 63) * 2 >> 4), za, kOf, i > 0 || d > 0);
                        }
                    commit(&sm.z_free[0]);
                }
                commit(&sm.s_full[n & 1]);
            };
            const auto sums = [&](int n) {
                if (kOne) fine = fine && barrier_wait(&sm.z_full[n & 1], (n >> 1) & 1);
                if (kHoldsRows && words != nullptr) fine = fine && barrier_wait(&sm.clean[n & 1], (n >> 1) & 1);
                fine = fine && barrier_wait(&sm.p_full[n & 1], (n >> 1) & 1);
                if (!fine) return;
                fence_after();
                const int run = n / kRun;
                if (n % kRun == 0) fine = barrier_wait(&sm.run_free, (run & 1) ^ 1);
                if (!fine) return;
                const uint32_t from = tmem + kScores + (kOne ? (n & 1) * kBuffer : 0), of = sums_of + (n & 1) * 3 * kTerm;
    #pragma unroll
                for (int i = 0; i < kPairs; ++i)
    #pragma unroll
                    for (int j = 0; j < kY; j += 16)
                        mma_ts<128>(tmem + kSums, from + 32 * left_term(i) + j / 2, of + right_term(i) * kTerm + (j * 128 >> 4), kAdd,
                                    n % kRun != 0 || i > 0 || j > 0);
                commit(kOne ? &sm.z_free[n & 1] : &sm.y_free[n & 1]);
                commit(&sm.done);
                if (n % kRun == kRun - 1 || n == count - 1) commit(&sm.run_full);
            };
            constexpr int kAhead = kOne ? 2 : 1;          // tiles whose scores are there before the first sums
            for (int n = 0; fine && n < count + kAhead; ++n) {
                if (n >= kAhead) sums(n - kAhead);
                if (fine && n < count) scores(n);
            }
            if (!fine) {          // (else the last run is waited for)
                commit(&sm.drained);
                barrier_wait(&sm.drained, 0);
            }
        } else if (warp == kLast + 2 && kHoldsRows && words != nullptr) {
            // rows of v (of k) that nobody may see: whatever they hold, their weight is 0 and has to stay it
            for (int n = 0; fine && n < count; ++n) {
                const uint32_t entry = tile_at(n);
                fine = barrier_wait(kOne ? &sm.z_full[n & 1] : &sm.y_full[n & 1], (n >> 1) & 1);
                if (fine && !(entry >> 31)) {
                    const uint2 see = __ldg(reinterpret_cast<const uint2 *>(words) + entry);
                    constexpr int kChunks = kD / 8;
                    for (int c = lane; c < kY * kChunks; c += 32) {
                        const int r = c / kChunks;
                        if (!(((r < 32 ? see.x : see.y) >> (r & 31)) & 1)) {
    #pragma unroll
                            for (int i = 0; i < 3; ++i)
                                *reinterpret_cast<uint4 *>((kOne ? sm.z[n & (kZ - 1)][i] : sm.y[n & 1][i]) + swizzled<kD, kY>(r, c % kChunks)) =
                                    make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_async_shared();
                }
                barrier_arrive(&sm.clean[n & 1]);
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

template <Mode M>
cudaError_t launch(const AttentionParams &p, const tc::TensorMap &y, const tc::TensorMap &z, cudaStream_t stream) {
    const auto kernel = attention_wide_kernel<M>;
    using Sh = Shape<M>;
    static std::atomic<bool> fits{false};
    if (!fits) fits = tc::registers_suffice(kernel, Sh::kThreads, 128 * (Sh::kGroups * Sh::kRegisters + Sh::kFew + Sh::kSumming));
    if (!fits) return cudaErrorInvalidConfiguration;
    constexpr size_t smem = sizeof(Shared<M>);
    static_assert(smem <= 227 * 1024);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const int64_t grid = (int64_t)p.B * p.K * p.splits * (((Shape<M>::kHoldsRows ? p.R : p.S) + kX - 1) / kX);
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return launch_dependent(kernel, dim3((unsigned)grid), Shape<M>::kThreads, smem, stream, p, y, z,
                            Shape<M>::kHoldsRows ? kY : kY / p.share * p.share);
}

bool make_state_maps(const AttentionParams &p, tc::TensorMap &k, tc::TensorMap &v) {
    const int64_t D8 = (p.D + 7) / 8 * 8, states[3] = {(int64_t)p.S * p.K * D8, p.K * D8, D8};
    return tc::make_map<__nv_bfloat16, kD>(k, p.k_terms, states, 3 * p.B, p.S, p.K, 1, (int)D8, kY) &&
           tc::make_map<__nv_bfloat16, kD>(v, p.v_terms, states, 3 * p.B, p.S, p.K, 1, (int)D8, kY);
}

}  // namespace

cudaError_t launch_attention_forward_wide(const AttentionParams &p, cudaStream_t stream) {
    tc::TensorMap k, v;
    if (!make_state_maps(p, k, v)) return cudaErrorNotSupported;
    const TermsParams terms = {{{p.k, p.k_terms, {p.ks[0], p.ks[1], p.ks[2]}, p.S, p.K}, {p.v, p.v_terms, {p.vs[0], p.vs[1], p.vs[2]}, p.S, p.K}},
                               2, p.B, p.D};
    const cudaError_t e = launch_attention_terms(terms, stream);
    return e == cudaSuccess ? launch<FORWARD>(p, k, v, stream) : e;
}

cudaError_t launch_attention_backward_wide(const AttentionParams &p, bool keys, cudaStream_t stream) {
    tc::TensorMap y, z;
    if (!keys) return make_state_maps(p, y, z) ? launch<ROWS>(p, y, z, stream) : cudaErrorNotSupported;
    const int64_t D8 = (p.D + 7) / 8 * 8, heads = (int64_t)p.K * p.share, rows[3] = {p.Q * heads * D8, heads * D8, D8};
    if (!tc::make_map<__nv_bfloat16, kD>(y, p.q_terms, rows, 3 * p.B, p.Q, p.K, p.share, (int)D8, kY) ||
        !tc::make_map<__nv_bfloat16, kD>(z, p.g_terms, rows, 3 * p.B, p.Q, p.K, p.share, (int)D8, kY))
        return cudaErrorNotSupported;
    const cudaError_t e = launch<VALUES>(p, y, z, stream);
    return e == cudaSuccess ? launch<KEYS>(p, y, z, stream) : e;
}

}  // namespace msda_b200
