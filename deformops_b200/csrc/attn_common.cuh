// Cross attention: what its kernels share.
//
// A call has B samples, K key heads and `share` query heads for each of them.  All queries that meet
// one (sample, key head) are the rows r = query * share + head of one matrix of R = Q * share rows,
// so that shared heads fill the same tiles and their gradients meet without atomics.
//
//   s = scale * q k^T      p = exp(s - max) / sum over the states that the row may see
//   o = p v                L = max + log(sum)      (kept, in base 2, for the backward pass)
//   dv = p^T do   dp = do v^T   ds = p (dp - rowsum(do o))   dq = scale ds k   dk = scale ds^T q
//
// A row that may see nothing has o = 0, L = +inf and no gradients (exp2(x - inf) = 0).
//
// Masks are packed into bits by kernels of their own (one pass over a byte mask that every head would
// otherwise read again): bit j % 32 of word j / 32 is set where state j may be seen; words behind the
// last state are 0.  `key_words` holds for every state whether any row may see it: the rows of k and v
// of states that nobody sees are never used, whatever they hold.  `lists` names the tiles of 64 and of 128
// states of which some may be seen, bit 31 set where all may: a pass over the states takes those and no
// others, and is split over CTAs by their number.
#pragma once

#include <type_traits>

#include "msda_common.cuh"

namespace msda_b200 {

constexpr int kMaskTile = 128;     // states per group of four mask words; mask rows are whole groups

struct AttentionParams {
    const void *q, *k, *v;
    const void *grad_out;                  // backward only, (B, Q, G * D) like `out`
    int64_t qs[3], ks[3], vs[3];           // strides of (sample, token, head) in elements
    int B, K, share, Q, S, R, D;
    float scale, scale_log2;               // scale * log2(e)
    const uint32_t *key_words;             // (B, key_word_heads, W) or null: every state may be seen
    const uint32_t *row_words;             // (B, row_word_heads, Q, W) or null: rows see what key_words has
    const uint32_t *lists;                 // (B, key_word_heads, 2 + T64 + T128): two counts, two lists; or null
    int key_word_heads, row_word_heads, W;
    void *out;                             // (B, Q, G * D)
    float *lse;                            // (B, K, R), log2 of the sum of exp2
    float *delta;                          // (B, K, R), rowsum(do o); backward only
    // float16: norms of do's rows, (B, K, R), 0 for rows that see nothing, and of v's, (B, K, S), 0 for states that nobody
    // sees; of every (sample, key head) the largest of the first, of |delta| and of the second
    float *row_norms, *state_norms;
    float4 *bounds, *bound_parts;          // and those of up to eight CTAs each, behind one another, where there are some
    int bound_ctas;
    void *dq, *dk, *dv;                    // contiguous (B, Q, G, D), (B, S, K, D)
    // work over the long axis is split into `splits` stretches of `tiles` tiles; with more than one,
    // partial results go to part (splits, B, K, rows, D) and part_lse (splits, B, K, rows)
    float *part, *part2, *part_lse;
    int splits, tiles;
    // float32 on the tensor cores: the operands' three bf16 terms, dense (3, B, tokens, heads, D8), D8 whole
    // vectors of eight channels
    void *q_terms, *k_terms, *v_terms, *g_terms;
};

// Float32 operands as x = x0 + x1 + x2 of bf16 (8 bits each), products x0 y0, x0 y1, x1 y0, x1 y1, x0 y2, x2 y0: what
// is left out is 2^-24 of a product.  In the order that has the small ones first.
constexpr int kPairs = 6;
__host__ __device__ constexpr int left_term(int pair) { return pair == 0 ? 2 : pair == 2 || pair == 3 ? 1 : 0; }
__host__ __device__ constexpr int right_term(int pair) { return pair == 1 ? 2 : pair == 2 || pair == 4 ? 1 : 0; }
// (x, y) as terms, packed like the products' operands
__device__ __forceinline__ void split_terms(float2 x, uint32_t (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        t[i] = VecTraits<__nv_bfloat16>::pack2(x);
        const float2 y = VecTraits<__nv_bfloat16>::unpack2(t[i]);
        x.x -= y.x, x.y -= y.y;
    }
}

// float16 has no normal numbers below 2^-14 and none above 65 504.  Weights, 1 / S or so where the softmax is flat, are
// multiplied by 2^8 before they are rounded for dv, which is divided by it.  dS is multiplied by a power of two of the row
// (of do, or of k and v) that a thread holds, which its sum is divided by: the one that brings a bound of |dP - delta| to
// 2^12 .. 2^13, so nothing can overflow and what is 2^-27 of the bound has all its bits still.  (Room is left for weights
// above 1: scores of 10^7 have an L that is rounded by more than 1, in base 2.)  The bound:
// |do_r v_j| <= |do_r| |v_j| with 2-norms, rows held with the largest |v| and the row's own delta, states held with the
// largest |do| and |delta| of the (sample, key head).  Rows of do that hold infinities or NaN do not count for the others.
// (Rows 2^-10 of the largest over 17 821 states: dq was 6.5 % off with one factor from the largest |do| of all.)
template <typename T>
constexpr bool kScaled = std::is_same_v<T, __half>;
constexpr float kWeightScale = 256.f, kWeightExponent = 8.f;
__device__ __forceinline__ float scale_below(float bound) {
    const uint32_t exponent = __float_as_uint(bound) >> 23;       // (bound < 2^(exponent - 126))
    return exponent >= 255 ? 1.f : __uint_as_float((266 - max(exponent, 64u)) << 23);
}
__device__ __forceinline__ float row_scale(const AttentionParams &p, int64_t bh, int r) {
    return scale_below(p.row_norms[bh * p.R + r] * p.bounds[bh].z + fabsf(p.delta[bh * p.R + r]));
}
__device__ __forceinline__ float state_scale(const AttentionParams &p, int64_t bh, int state) {
    const float4 most = p.bounds[bh];
    return scale_below(most.x * p.state_norms[bh * p.S + state] + most.y);
}

// ---- which states a tile of 32 * N of them may use --------------------------------------------------
__device__ __forceinline__ const uint32_t *key_words_of(const AttentionParams &p, int b, int h) {
    if (p.key_words == nullptr) return nullptr;
    return p.key_words + ((int64_t)b * p.key_word_heads + (p.key_word_heads > 1 ? h : 0)) * p.W;
}

// word `w` of the states of a (sample, head): those that exist where there is no mask
__device__ __forceinline__ uint32_t key_word(const uint32_t *words, int S, int w) {
    if (words != nullptr) return __ldg(words + w);
    const int left = S - 32 * w;
    return left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1;
}

// ---- the tiles of BN states that a stretch of a pass takes -----------------------------------------
__host__ __device__ inline int64_t list_words(int64_t S) { return (2 + (S + 63) / 64 + (S + 127) / 128 + 3) / 4 * 4; }

template <int BN>
struct Tiles {
    const uint32_t *list;        // entries from the first one on, or null: all tiles
    int first, count, S;

    __device__ __forceinline__ Tiles(const AttentionParams &p, int b, int h, int part) : list(nullptr), S(p.S) {
        int all = (S + BN - 1) / BN;
        if (p.lists != nullptr) {
            const uint32_t *l = p.lists + ((int64_t)b * p.key_word_heads + (p.key_word_heads > 1 ? h : 0)) * list_words(S);
            all = (int)__ldg(l + (BN == 128));
            list = l + 2 + (BN == 128 ? (S + 63) / 64 : 0);
        }
        stretch(all, p.splits, part, first, count);
        if (list != nullptr) list += first;
    }
    // the part-th of `splits` nearly equal stretches
    static __device__ __forceinline__ void stretch(int all, int splits, int part, int &first, int &count) {
        const int each = all / splits, more = all - each * splits;
        first = part * each + min(part, more);
        count = each + (part < more);
    }
    // tile n of the stretch, bit 31 set where all of its states may be seen (by somebody)
    __device__ __forceinline__ uint32_t operator[](int n) const {
        if (list != nullptr) return __ldg(list + n);
        return (uint32_t)(first + n) | ((first + n + 1) * (int64_t)BN <= S ? 0x80000000u : 0u);
    }
};

// the mask words of packed row r, or null where rows have none of their own
__device__ __forceinline__ const uint32_t *row_words_of(const AttentionParams &p, int b, int h, int r) {
    if (p.row_words == nullptr) return nullptr;
    const int query = r / p.share;
    const int64_t head = p.row_word_heads > 1 ? (int64_t)h * p.share + (r - query * p.share) : 0;
    return p.row_words + (((int64_t)b * p.row_word_heads + head) * p.Q + query) * p.W;
}

// element offset of packed row r of sample b, key head h in a (B, Q, G, D) tensor of these strides
__device__ __forceinline__ int64_t row_offset(const int64_t (&s)[3], int share, int b, int h, int r) {
    const int query = share == 1 ? r : r / share;
    const int head = h * share + (r - query * share);
    return b * s[0] + query * s[1] + head * s[2];
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a * b + c of pairs, into registers of its own
__device__ __forceinline__ float2 fma2(const float2 a, const float2 b, const float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)),
          "l"(reinterpret_cast<const unsigned long long &>(c)));
    return r;
}
__device__ __forceinline__ float2 add2(const float2 a, const float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
    return r;
}

// ---- host side ------------------------------------------------------------------------------------
// A launch that may become resident while the kernel before it drains; it begins with grid_dependency_wait().  For
// the small kernels of a call, each of which would wait for the one before to leave the GPU.
template <typename... Formal, typename... Actual>
inline cudaError_t launch_dependent(void (*kernel)(Formal...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                                    const Actual &...actual) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(actual)...);
}

// 16-bit types, and float32 of up to 64 channels with its terms; row_tiles of 128 rows to a CTA (0: a small
// CTA of 128 rows), stretches of whole tiles of 64 states (128 of 16 bits where D > 64, but for small CTAs).
// cudaErrorNotSupported (and nothing launched) where an operand cannot be described to TMA.  Backward: at most 64 query
// heads to a key head.
cudaError_t launch_attention_forward_tc(const AttentionParams &p, int dtype, int row_tiles, cudaStream_t stream);
// float32 of 65 to 128 channels, the same way (backward: of a pass over the held states both gradients)
cudaError_t launch_attention_forward_wide(const AttentionParams &p, cudaStream_t stream);
cudaError_t launch_attention_backward_wide(const AttentionParams &p, bool keys, cudaStream_t stream);
// at most 16 rows to a key head; stretches of p.tiles blocks
struct FewShape {
    int block, resident;      // states of a block; CTAs to an SM
};
FewShape attention_few_shape(int dtype, int64_t D, int64_t rows);
cudaError_t launch_attention_few(const AttentionParams &p, int dtype, cudaStream_t stream);
cudaError_t launch_attention_backward_tc(const AttentionParams &p, int dtype, bool keys, cudaStream_t stream);
// the same for more of them
cudaError_t launch_attention_backward_mma(const AttentionParams &p, int dtype, bool keys, cudaStream_t stream);

// the terms of (B, tokens, heads, D) float32 tensors
struct TermsParams {
    struct Tensor {
        const void *x;
        void *terms;
        int64_t strides[3];
        int tokens, heads;
    } of[4];
    int tensors, B, D;
};
cudaError_t launch_attention_terms(const TermsParams &p, cudaStream_t stream);
cudaError_t launch_attention_delta(const AttentionParams &p, int dtype, cudaStream_t stream);
// parts of a split pass to the result: outputs and sums (forward), or the sum of gradients
cudaError_t launch_attention_join(const AttentionParams &p, int dtype, cudaStream_t stream);
cudaError_t launch_attention_sum(const AttentionParams &p, bool keys, int dtype, cudaStream_t stream);
struct MaskParams {
    const uint8_t *padding, *mask;        // true: not to be seen; either may be null
    int64_t ps[2], ms[4];                 // strides of (sample, state), (sample, head, query, state)
    int B, H, KW, Q, S, W;                // H heads of the mask (0: none), KW heads of the key words
    uint32_t *key_words, *row_words, *lists;
};
cudaError_t launch_attention_mask(const MaskParams &p, cudaStream_t stream);

}  // namespace msda_b200
