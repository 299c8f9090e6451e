// C ABI of cross attention (declared in include/msda_b200.h): argument checks and the plan of a call.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "../../include/msda_b200.h"
#include "attn_common.cuh"

namespace msda_b200 {

namespace {

// how a pass over the tiles of the long axis is split: stretches, tiles of each
struct AttentionSplit {
    int splits, tiles;
};

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int refuse(int status, const char *message) { return set_last_error(status, message); }

int64_t mask_words(int64_t states) { return (states + kMaskTile - 1) / kMaskTile * 4; }

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// one pass of a call: its split, and the bytes that its parts take
struct Pass {
    AttentionSplit split;
    int64_t bytes;       // parts
    bool tensor_cores;
    int row_tiles;       // forward: tiles of 128 rows that a CTA holds, 0 for a small one
};

// What a pass takes, in twentieths of a tile of 256 rows: an SM takes `at_once` items together, each of them a share
// of the time of all, which has its tiles, a beginning and an end, and parts to write and read where it is split.
struct Cost {
    int64_t tile, item, join, at_once;
};

// Of `fewest` to `most` stretches of `tiles` tiles the number that cost(stretches, tiles of each) has lowest: all small
// numbers, a few of the larger ones, and `full`, with which the GPU is just full.
template <typename F>
AttentionSplit best_split(int64_t tiles, int64_t fewest, int64_t most, int64_t full, const F &cost, int64_t *best_cost = nullptr) {
    int64_t best = fewest, lowest = INT64_MAX;
    const auto consider = [&](int64_t s) {
        const int64_t all = cost(s, (tiles + s - 1) / s);
        if (all < lowest) best = s, lowest = all;
    };
    for (int64_t s = fewest; s <= std::max(fewest, most); s += 1 + s / 16) consider(s);
    if (full > fewest && full <= most) consider(full);
    if (best_cost != nullptr) *best_cost = lowest;
    const int64_t each = std::max<int64_t>(1, (tiles + best - 1) / best);
    return {(int)std::max<int64_t>(1, (tiles + each - 1) / each), (int)each};
}

// the number of splits that ends soonest, with items of at most `most` tiles
AttentionSplit even_split(int64_t items, int64_t tiles, const Cost &cost, int64_t most, int64_t *best_cost = nullptr) {
    const int64_t at_once = 148 * cost.at_once;
    return best_split(tiles, std::max<int64_t>(1, (tiles + most - 1) / most), std::min({tiles / 2, at_once, at_once * 8 / items + 1}), at_once / items,
                      [&](int64_t s, int64_t each) {
                          return std::max(cost.at_once, (items * s + 147) / 148) * (each * cost.tile + cost.item + (s > 1 ? cost.join : 0)) +
                                 (s > 1 ? 80 : 0);
                      },
                      best_cost);
}

// The same where `slots` CTAs of four warps run at a time, whatever else does: a stretch takes its blocks and about 8
// more, parts 16 and some to join.  Four parts for 512 (sample, head)s of 4000 states of 64 channels are 89 us where one
// is 97 (only 512 of 740 slots have work), for 512 of 8000 of 128 channels 340 us and 464 (444 slots); 18 for 8 of
// 1500 states 6.2 us, one 15.2; one for 8 of 77 states 3.3 us, two 5.0.
AttentionSplit few_split(int64_t items, int64_t blocks, int64_t slots) {
    return best_split(blocks, 1, std::min(blocks / 4, slots * 8 / items + 1), slots / items, [&](int64_t s, int64_t each) {
        return (items * s + slots - 1) / slots * (each + 8) + (s > 1 ? 16 + s / 4 : 0);
    });
}

// Float32 sums on the tensor cores are cut off, not rounded, at every product that is added to them.  The kernels take
// them on after a few tiles, but for two forms of the forward pass up to 32 channels (one row tile, small CTAs), whose groups
// have at most eight (over 32 the result was 1.1e-5 off, relative; over eight it is 3e-6).
constexpr int64_t kMostTiles = 1 << 30, kMostFloatTiles = 8;
constexpr int64_t kFewRows = 16;
constexpr float kLog2e = 1.4426950408889634f;

bool wide_float(const msda_b200_attention &c) { return c.dtype == MSDA_B200_F32 && c.head_dim > 64; }

// The forward pass has three forms of CTA: two tiles of 128 rows; one, with twice the groups to it; or, where a
// pass is short, small ones of 128 rows, several to an SM, that begin and end in one another's shadow.  The costs
// are fits of times (0.7 us for 20 with up to 64 channels, 2 us with 128).  bf16, 4096 rows of 32 heads of 64: small ones
// 20.7 us over 77 states and 205 over 4096, big ones 31.3 and 265 (in two parts; 214 in one); 1 x 16 384 x 16 heads
// over 4096: big 361 us, small 399; 64 heads of 100 rows over 17 821 states: one tile to a CTA 61 us, small 84.
// float32, heads of 32: 2 x 8 heads of 300 rows over 17 821 states, one tile to a CTA 130 us, two 143; 4 heads of 8192 rows over
// 4096, two 105 us (137 in four short parts).
void plan_forward(const msda_b200_attention &c, int64_t rows, Pass &pass) {
    const int64_t bk = c.batch * c.kv_heads;
    const bool half = c.dtype != MSDA_B200_F32, wide = wide_float(c), deep = c.head_dim > 64 && !wide;
    const int64_t tiles = (c.states + 63) / 64, big = deep ? (c.states + 127) / 128 : tiles, one = (rows + 127) / 128, two = (rows + 255) / 256;
    const bool runs = half || c.head_dim > 32;
    int64_t lowest = INT64_MAX;
    // `groups` with sums of their own share a part.  Parts that are short for the sums' sake have theirs in the workspace:
    // no more of them than eight rounds of CTAs would make of the rows anyway.
    const auto take = [&](int row_tiles, int64_t items, int64_t of, const Cost &cost, int groups) {
        const int64_t most = runs || row_tiles == 2 ? kMostTiles : kMostFloatTiles * groups, fewest = (of + most - 1) / most;
        if (fewest > 1 && fewest * items > 148 * 8 * cost.at_once) return;
        int64_t all;
        const AttentionSplit split = even_split(items, of, cost, most, &all);
        if (all < lowest) lowest = all, pass.split = split, pass.row_tiles = row_tiles;
    };
    take(1, bk * one, big, {deep || !half ? 13 : 11, deep ? 50 : half ? 150 : 100, 30, 1}, 4);
    if (wide) return;
    take(2, bk * two, big, {runs ? 20 : 22, deep ? 80 : half ? 190 : 125, 60, 1}, 2);
    if (deep) take(0, bk * one, tiles, {7, 40, 30, 2}, 1);
    else if (half || c.head_dim <= 32) take(0, bk * one, tiles, {half ? 13 : 11, 50, 30, 3}, 1);
}

Pass forward_pass(const msda_b200_attention &c) {
    const int64_t rows = c.queries * (c.heads / c.kv_heads), bk = c.batch * c.kv_heads;
    Pass pass{};
    if (rows > kFewRows) {
        pass.tensor_cores = true;
        plan_forward(c, rows, pass);
    } else {
        const FewShape few = attention_few_shape(c.dtype, c.head_dim, rows);
        pass.split = few_split(bk, (c.states + few.block - 1) / few.block, 148 * few.resident);
    }
    const int64_t parts = pass.split.splits * bk * rows;
    pass.bytes = pass.split.splits > 1 ? round16(parts * 4) + parts * c.head_dim * 4 : 0;
    return pass;
}

Pass backward_pass(const msda_b200_attention &c, bool keys) {
    const int64_t share = c.heads / c.kv_heads, rows = c.queries * share, bk = c.batch * c.kv_heads;
    const int64_t held = keys ? c.states : rows, walked = keys ? rows : c.states;
    Pass pass{};
    if (share <= 64) {
        pass.tensor_cores = true;
        const int64_t x_rows = keys || wide_float(c) ? 128 : 128 / share * share, y_rows = keys ? 64 / share * share : 64;
        pass.split = even_split(bk * ((held + x_rows - 1) / x_rows), (walked + y_rows - 1) / y_rows, {20, 120, 60, 1}, kMostTiles);
    } else {
        const int tile = c.head_dim > 64 ? 32 : 64;
        pass.split = few_split(bk * ((held + 63) / 64), (walked + tile - 1) / tile, 148 * 3);
    }
    pass.bytes = pass.split.splits > 1 ? (keys ? 2 : 1) * pass.split.splits * bk * held * c.head_dim * 4 : 0;
    return pass;
}

cudaError_t launch_backward(AttentionParams &p, const Pass &pass, int dtype, bool keys, cudaStream_t stream) {
    p.splits = pass.split.splits, p.tiles = pass.split.tiles;
    if (!pass.tensor_cores) return launch_attention_backward_mma(p, dtype, keys, stream);
    return dtype == MSDA_B200_F32 && p.D > 64 ? launch_attention_backward_wide(p, keys, stream)
                                              : launch_attention_backward_tc(p, dtype, keys, stream);
}

// the terms of `tokens` x `heads` float32 rows, where a pass needs them
int64_t term_bytes(const msda_b200_attention &c, int64_t tokens, int64_t heads) {
    return 6 * c.batch * tokens * heads * ((c.head_dim + 7) / 8 * 8);
}
int64_t forward_bytes(const msda_b200_attention &c, const Pass &pass) {
    const bool terms = c.dtype == MSDA_B200_F32 && pass.tensor_cores;
    return round16(pass.bytes) + (terms ? 2 * term_bytes(c, c.states, c.kv_heads) : 0);
}
// rowsum(do o), and behind it what float16 is scaled by: norms of the rows and of the states, bounds
int64_t delta_bytes(const msda_b200_attention &c) { return round16(c.batch * c.heads * c.queries * 4); }
int64_t state_norm_bytes(const msda_b200_attention &c) { return round16(c.batch * c.kv_heads * c.states * 4); }
int64_t bound_ctas(const msda_b200_attention &c) {
    return std::min<int64_t>(8, (std::max(c.queries * (c.heads / c.kv_heads), c.states) + 16383) / 16384);
}
int64_t scaling_bytes(const msda_b200_attention &c) {
    return c.dtype == MSDA_B200_F16 ? delta_bytes(c) + state_norm_bytes(c) + c.batch * c.kv_heads * (1 + bound_ctas(c)) * 16 : 0;
}

int64_t backward_bytes(const msda_b200_attention &c, const Pass &keys, const Pass &rows) {
    const bool terms = c.dtype == MSDA_B200_F32 && keys.tensor_cores;
    return delta_bytes(c) + scaling_bytes(c) + round16(std::max(keys.bytes, rows.bytes)) +
           (terms ? 2 * term_bytes(c, c.states, c.kv_heads) + 2 * term_bytes(c, c.queries, c.heads) : 0);
}

int check(const msda_b200_attention *c) {
    if (c == nullptr) return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: null call");
    if (c->dtype != MSDA_B200_F32 && c->dtype != MSDA_B200_F16 && c->dtype != MSDA_B200_BF16)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: dtype is not f32, f16 or bf16");
    if (c->batch < 0 || c->queries < 0 || c->states < 0 || c->heads <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: sizes out of range");
    if (c->heads % c->kv_heads != 0)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: heads must be a multiple of kv_heads");
    const int vec = c->dtype == MSDA_B200_F32 ? 4 : 8;
    if (c->head_dim % vec != 0 || c->head_dim > 128)
        return refuse(MSDA_B200_UNSUPPORTED, "attention: head_dim must be whole 16-byte vectors and at most 128");
    constexpr int64_t kMost = (int64_t)1 << 30;
    if (c->batch > kMost || c->heads > kMost || c->batch * c->heads > 1 << 20 || c->queries > kMost ||
        c->states > kMost || c->queries * (c->heads / c->kv_heads) > kMost)
        return refuse(MSDA_B200_UNSUPPORTED, "attention: more than 2^30 rows or states, or 2^20 heads of all samples");
    if (!(c->scale > 0.f) || std::isinf(c->scale * kLog2e))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: scale must be positive and finite, times log2(e) too");
    if (c->mask_heads != 0 && c->mask_heads != 1 && c->mask_heads != c->heads)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: mask_heads must be 0, 1 or heads");
    if (!aligned16(c->mask)) return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: misaligned mask");
    for (const int64_t *s : {c->query_strides, c->key_strides, c->value_strides})
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0 || s[i] % vec != 0)
                return refuse(MSDA_B200_INVALID_ARGUMENT, "attention: strides must be whole 16-byte vectors");
    if ((c->queries > 1 && c->query_strides[1] == 0) || (c->states > 1 && (c->key_strides[1] == 0 || c->value_strides[1] == 0)) ||
        (c->heads > c->kv_heads && c->query_strides[2] == 0))
        return refuse(MSDA_B200_UNSUPPORTED, "attention: tokens, and query heads that share a key head, need strides of their own");
    return MSDA_B200_OK;
}

AttentionParams params(const msda_b200_attention &c, const void *q, const void *k, const void *v) {
    AttentionParams p{};
    p.q = q, p.k = k, p.v = v;
    for (int i = 0; i < 3; ++i) p.qs[i] = c.query_strides[i], p.ks[i] = c.key_strides[i], p.vs[i] = c.value_strides[i];
    p.B = (int)c.batch, p.K = (int)c.kv_heads, p.share = (int)(c.heads / c.kv_heads), p.Q = (int)c.queries;
    p.S = (int)c.states, p.R = p.Q * p.share, p.D = (int)c.head_dim;
    p.scale = c.scale;
    p.scale_log2 = c.scale * kLog2e;
    p.W = (int)mask_words(c.states);
    if (c.mask != nullptr) {
        p.lists = static_cast<const uint32_t *>(c.mask);
        p.key_word_heads = c.mask_heads > 1 ? p.K : 1;
        p.key_words = p.lists + (int64_t)p.B * p.key_word_heads * list_words(p.S);
        if (c.mask_heads > 0) {
            p.row_words = p.key_words + (int64_t)p.B * p.key_word_heads * p.W;
            p.row_word_heads = c.mask_heads;
        }
    }
    return p;
}

int status_of(cudaError_t e) {
    return e == cudaSuccess ? MSDA_B200_OK : refuse(MSDA_B200_CUDA_ERROR, cudaGetErrorString(e));
}

}  // namespace

}  // namespace msda_b200

extern "C" {

using namespace msda_b200;

int64_t msda_b200_attention_mask_bytes(int64_t batch, int64_t queries, int64_t states, int64_t kv_heads,
                                       int mask_heads) {
    if (batch <= 0 || queries < 0 || states < 0 || kv_heads <= 0 || mask_heads < 0) return 0;
    const int64_t key_heads = mask_heads > 1 ? kv_heads : 1;
    return 4 * batch * (key_heads * list_words(states) + mask_words(states) * (key_heads + mask_heads * queries));
}

int msda_b200_attention_pack_mask(const void *padding, const int64_t *padding_strides, const void *mask,
                                  const int64_t *mask_strides, int mask_heads, int64_t batch, int64_t queries,
                                  int64_t states, int64_t kv_heads, void *packed, int device, void *stream) {
    if (batch < 0 || queries < 0 || states < 0 || kv_heads <= 0 || mask_heads < 0 || (mask == nullptr) != (mask_heads == 0) ||
        (mask_heads > 1 && mask_heads % kv_heads != 0))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_pack_mask: sizes out of range");
    if ((padding == nullptr && mask == nullptr) || (padding != nullptr && padding_strides == nullptr) ||
        (mask != nullptr && mask_strides == nullptr) || packed == nullptr || !aligned16(packed))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_pack_mask: null or misaligned pointer");
    if (batch > 1 << 20 || queries > 1 << 30 || states > 1 << 30 || mask_heads > 1 << 20)
        return refuse(MSDA_B200_UNSUPPORTED, "attention_pack_mask: sizes too large");
    if (batch == 0 || states == 0 || (mask != nullptr && queries == 0)) return MSDA_B200_OK;
    MaskParams p{};
    p.padding = static_cast<const uint8_t *>(padding), p.mask = static_cast<const uint8_t *>(mask);
    for (int i = 0; i < 2 && padding != nullptr; ++i) p.ps[i] = padding_strides[i];
    for (int i = 0; i < 4 && mask != nullptr; ++i) p.ms[i] = mask_strides[i];
    p.B = (int)batch, p.H = mask_heads, p.KW = mask_heads > 1 ? (int)kv_heads : 1, p.Q = (int)queries;
    p.S = (int)states, p.W = (int)mask_words(states);
    p.lists = static_cast<uint32_t *>(packed);
    p.key_words = p.lists + (int64_t)p.B * p.KW * list_words(states);
    p.row_words = p.key_words + (int64_t)p.B * p.KW * p.W;
    const DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return status_of(guard.err);
    const cudaError_t e = launch_attention_mask(p, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) count_launches(mask != nullptr ? 3 : 1, 0);
    return status_of(e);
}

int64_t msda_b200_attention_workspace_bytes(const msda_b200_attention *call, int backward) {
    if (check(call) != MSDA_B200_OK || call->batch == 0 || call->queries == 0 || call->states == 0) return 0;
    if (!backward) return forward_bytes(*call, forward_pass(*call));
    return backward_bytes(*call, backward_pass(*call, true), backward_pass(*call, false));
}

int msda_b200_attention_forward(const msda_b200_attention *call, const void *query, const void *key, const void *value,
                                void *out, float *lse, void *workspace, int64_t workspace_bytes, int device,
                                void *stream) {
    const int st = check(call);
    if (st != MSDA_B200_OK) return st;
    if (call->batch == 0 || call->queries == 0) return MSDA_B200_OK;
    if (out == nullptr || lse == nullptr || !aligned16(out) || !aligned16(lse))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_forward: null or misaligned output");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return status_of(guard.err);
    if (call->states == 0) {        // nothing to see: zeros (and L, which no backward pass will read)
        const int64_t n = call->batch * call->queries * call->heads * call->head_dim;
        count_launches(0, 1);
        return status_of(cudaMemsetAsync(out, 0, n * (call->dtype == MSDA_B200_F32 ? 4 : 2), s));
    }
    if (query == nullptr || key == nullptr || value == nullptr || !aligned16(query) || !aligned16(key) || !aligned16(value))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_forward: null or misaligned operand");
    const Pass pass = forward_pass(*call);
    const int64_t needed = forward_bytes(*call, pass);
    if (needed > workspace_bytes || (needed > 0 && (workspace == nullptr || !aligned16(workspace))))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_forward: workspace too small or misaligned");
    AttentionParams p = params(*call, query, key, value);
    p.out = out, p.lse = lse;
    p.splits = pass.split.splits, p.tiles = pass.split.tiles;
    p.part_lse = static_cast<float *>(workspace);
    p.part = p.part_lse + round16((int64_t)p.splits * p.B * p.K * p.R * 4) / 4;
    p.k_terms = static_cast<char *>(workspace) + round16(pass.bytes);
    p.v_terms = static_cast<char *>(p.k_terms) + term_bytes(*call, call->states, call->kv_heads);
    const int terms = call->dtype == MSDA_B200_F32 && pass.tensor_cores ? 1 : 0;
    cudaError_t e = !pass.tensor_cores ? launch_attention_few(p, call->dtype, s)
                    : wide_float(*call) ? launch_attention_forward_wide(p, s)
                                        : launch_attention_forward_tc(p, call->dtype, pass.row_tiles, s);
    if (e == cudaSuccess && p.splits > 1) e = launch_attention_join(p, call->dtype, s);
    if (e == cudaSuccess) count_launches((p.splits > 1 ? 2 : 1) + terms, 0);
    return status_of(e);
}

int msda_b200_attention_backward(const msda_b200_attention *call, const void *query, const void *key, const void *value,
                                 const void *out, const void *grad_out, const float *lse, void *grad_query,
                                 void *grad_key, void *grad_value, void *workspace, int64_t workspace_bytes, int device,
                                 void *stream) {
    const int st = check(call);
    if (st != MSDA_B200_OK) return st;
    if (call->batch == 0) return MSDA_B200_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return status_of(guard.err);
    const int64_t e_size = call->dtype == MSDA_B200_F32 ? 4 : 2;
    const int64_t row_bytes = call->batch * call->queries * call->heads * call->head_dim * e_size;
    const int64_t state_bytes = call->batch * call->states * call->kv_heads * call->head_dim * e_size;
    for (const void *x : {grad_query, grad_key, grad_value})
        if (!aligned16(x)) return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_backward: misaligned gradient");
    if ((row_bytes > 0 && grad_query == nullptr) || (state_bytes > 0 && (grad_key == nullptr || grad_value == nullptr)))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_backward: null gradient");
    if (row_bytes == 0 || state_bytes == 0) {
        cudaError_t e = cudaSuccess;
        if (row_bytes > 0) e = cudaMemsetAsync(grad_query, 0, row_bytes, s);
        if (e == cudaSuccess && state_bytes > 0) e = cudaMemsetAsync(grad_key, 0, state_bytes, s);
        if (e == cudaSuccess && state_bytes > 0) e = cudaMemsetAsync(grad_value, 0, state_bytes, s);
        if (e == cudaSuccess) count_launches(0, (row_bytes > 0) + 2 * (state_bytes > 0));
        return status_of(e);
    }
    for (const void *x : {query, key, value, out, grad_out, (const void *)lse, (const void *)workspace})
        if (x == nullptr || !aligned16(x))
            return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_backward: null or misaligned operand");
    const Pass keys = backward_pass(*call, true), rows = backward_pass(*call, false);
    if (backward_bytes(*call, keys, rows) > workspace_bytes)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "attention_backward: workspace too small");
    AttentionParams p = params(*call, query, key, value);
    p.out = const_cast<void *>(out), p.grad_out = grad_out, p.lse = const_cast<float *>(lse);
    p.dq = grad_query, p.dk = grad_key, p.dv = grad_value;
    p.delta = static_cast<float *>(workspace);
    p.row_norms = p.delta + delta_bytes(*call) / 4;
    p.state_norms = p.row_norms + delta_bytes(*call) / 4;
    p.bounds = reinterpret_cast<float4 *>(p.state_norms + state_norm_bytes(*call) / 4);
    p.bound_parts = p.bounds + call->batch * call->kv_heads;
    p.bound_ctas = (int)bound_ctas(*call);
    p.part = p.delta + (delta_bytes(*call) + scaling_bytes(*call)) / 4;
    int launches = call->dtype != MSDA_B200_F16 ? 3 : p.bound_ctas > 1 ? 5 : 4;
    cudaError_t e = launch_attention_delta(p, call->dtype, s);
    if (call->dtype == MSDA_B200_F32 && keys.tensor_cores) {
        const int64_t gs[3] = {call->queries * call->heads * call->head_dim, call->heads * call->head_dim, call->head_dim};
        char *terms = reinterpret_cast<char *>(p.part) + round16(std::max(keys.bytes, rows.bytes));
        const int64_t state_terms = term_bytes(*call, call->states, call->kv_heads), row_terms = term_bytes(*call, call->queries, call->heads);
        p.k_terms = terms, p.v_terms = terms + state_terms, p.q_terms = terms + 2 * state_terms;
        p.g_terms = terms + 2 * state_terms + row_terms;
        const int H = (int)call->heads;
        const TermsParams all = {{{p.k, p.k_terms, {p.ks[0], p.ks[1], p.ks[2]}, p.S, p.K},
                                  {p.v, p.v_terms, {p.vs[0], p.vs[1], p.vs[2]}, p.S, p.K},
                                  {p.q, p.q_terms, {p.qs[0], p.qs[1], p.qs[2]}, p.Q, H},
                                  {p.grad_out, p.g_terms, {gs[0], gs[1], gs[2]}, p.Q, H}},
                                 4, p.B, p.D};
        if (e == cudaSuccess) e = launch_attention_terms(all, s);
        ++launches;
    }
    if (e == cudaSuccess) {
        p.part2 = p.part + (int64_t)keys.split.splits * p.B * p.K * p.S * p.D;
        e = launch_backward(p, keys, call->dtype, true, s);
        if (e == cudaSuccess && p.splits > 1) e = launch_attention_sum(p, true, call->dtype, s);
        launches += (p.splits > 1) + (wide_float(*call) && keys.tensor_cores);
    }
    if (e == cudaSuccess) {
        e = launch_backward(p, rows, call->dtype, false, s);
        if (e == cudaSuccess && p.splits > 1) e = launch_attention_sum(p, false, call->dtype, s);
        launches += p.splits > 1;
    }
    if (e == cudaSuccess) count_launches(launches, 0);
    return status_of(e);
}

}  // extern "C"
