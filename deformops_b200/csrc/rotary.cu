// Rotary positions of several axes: pairs of channels turned by position * frequency.
//
//   (a, b) -> (a cos - b sin, a sin + b cos),   angle = position of the pair's axis * its frequency
//
// One pass over x, bound by its bytes.  A CTA takes a few tokens of a sample: its threads ask for the vectors that
// they will turn (both halves of the pairs), form the sine and cosine of every (token, pair) once for all heads
// while those are on their way, and turn them.  Angles are turns in more than 32 bits, reduced to [-1/2, 1/2] before
// anything is rounded: at position 10^6 a 32-bit angle is 0.03 off.  float32 positions of less than 2^20 turns take a
// frequency of two floats and the rounding error of the product that a fused multiply-add gives (2^-48 of the turns),
// all others float64.  (Rounding to whole turns by two additions: with rint and the branch this costs 20.5 us, below.)
// The frequencies go to shared memory first: lanes that index kernel parameters differently are served one by one.
// The backward pass is the same kernel with the angles' sign turned.
//
// 4 x 21 504 tokens of 8 heads of 32, bf16: 17.5 us (5.0 TB/s; 19.3 with divisions and without packed arithmetic, when
// instructions filled 76 % of the issue slots); 2 x 16 384 of 16 heads of 128, float16, 44 us (6.1 TB/s); 2 x 17 821 of 8
// heads of 32, float32, 14 us (5.3 TB/s).
#include <algorithm>
#include <type_traits>

#include "../../include/msda_b200.h"
#include "msda_common.cuh"

namespace msda_b200 {

namespace {

constexpr int kThreads = 128;
constexpr int kMostPairs = 128;
constexpr int kInFlight = 2;          // pairs of vectors that a thread asks for at a time
constexpr float kFarTurns = 1048576.f;

struct RotaryParams {
    const void *x, *positions;
    void *out;
    int64_t xs[3], ps[3];                 // strides of (sample, token, head), (sample, token, axis)
    int N, G, D, pairs, tile;             // tile: tokens of a CTA
    unsigned tiles;                       // of a sample
    // How a CTA's threads go through its tokens' units (vectors, or pairs of them) and pairs.  Divisions are the host's:
    // a thread has two units, and would spend a third of its instructions on them.
    int units, turning, per_token;        // units of a head, those that turn, units of a token
    int tokens, heads, step;              // from a thread's unit to its next one
    int pair_tokens, pair_step;           // the same of pairs
    float per_token_inverse, units_inverse, pairs_inverse;
    int position_dtype;
    float sign;
    double turns[kMostPairs];             // frequency / 2 pi
    uint8_t axis[kMostPairs];
};

__device__ __forceinline__ double position(const RotaryParams &p, int64_t at) {
    switch (p.position_dtype) {
        case MSDA_B200_F64: return __ldg(static_cast<const double *>(p.positions) + at);
        case MSDA_B200_I32: return __ldg(static_cast<const int *>(p.positions) + at);
        default: return (double)__ldg(static_cast<const long long *>(p.positions) + at);
    }
}

// t / n of a thread's number t, given 1 / n: t + 1/2 is 1/2 away from every multiple of n, a rounding 2^-17 at most
__device__ __forceinline__ int over(int t, float inverse) { return (int)(((float)t + 0.5f) * inverse); }

// the whole number that is nearest to x, |x| < 2^22
__device__ __forceinline__ float nearest(float x) { return __fadd_rn(__fadd_rn(x, 12582912.f), -12582912.f); }

__device__ __forceinline__ float far_turns(double at, double frequency) {
    const double all = at * frequency;
    return (float)(all - rint(all));
}

// (a, b) turned; written out, so that every variant of the kernel gives the same bits
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = __fmaf_rn(a, c, __fmul_rn(-b, s));
    b = __fmaf_rn(a, s, __fmul_rn(b, c));
    a = x;
}

// the same of two pairs
__device__ __forceinline__ void turn2(float2 &a, float2 &b, float2 c, float2 s) {
    float2 x = fmul2(b, make_float2(-s.x, -s.y)), y = fmul2(b, c);
    ffma2(x, a, c), ffma2(y, a, s);
    a = x, b = y;
}

// Sine and cosine of so many turns, |turns| <= 1/2.  Results of 16 bits have a half step of 2^-11 and more, where
// the hardware's approximation (2^-20 within half a turn) costs 6 instructions instead of 50.
template <typename T>
__device__ __forceinline__ void sine_cosine(float turns, float &s, float &c) {
    if constexpr (sizeof(T) == 4) {
        sincospif(2.f * turns, &s, &c);
    } else {
        const float x = 6.283185307f * turns;
        s = __sinf(x), c = __cosf(x);
    }
}

// WIDE: 16-byte vectors, else single elements; INTERLEAVED: a pair is two neighbours, else the channels i and
// i + pairs.  The table has the cosines of a token's pairs, then their sines.
template <typename T, bool WIDE, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int VEC = WIDE ? 16 / sizeof(T) : 1;
    using Raw = std::conditional_t<WIDE, uint4, T>;
    // a unit: two vectors of pairs (one of interleaved pairs where it is wide), or one behind the turned channels
    constexpr bool kOne = INTERLEAVED && WIDE;
    constexpr int kUnits = kOne ? 2 * kInFlight : kInFlight;
    extern __shared__ __align__(16) float table[];
    __shared__ double frequency[kMostPairs];
    __shared__ float2 split[kMostPairs];
    __shared__ int axis[kMostPairs];
    const unsigned b = blockIdx.x / p.tiles;
    const int first = (int)(blockIdx.x - b * p.tiles) * p.tile, count = min(p.tile, p.N - first);
    const int turning = p.turning, units = p.units, per_token = p.per_token, all = count * per_token;
    // this thread's next unit, and how far the one after that is
    int token = over(threadIdx.x, p.per_token_inverse), head = over(threadIdx.x - token * per_token, p.units_inverse);
    int unit = threadIdx.x - token * per_token - head * units;
    const T *const x = static_cast<const T *>(p.x) + b * p.xs[0] + first * p.xs[1];
    T *const out = static_cast<T *>(p.out) + ((int64_t)b * p.N + first) * p.G * p.D;
    const int other = INTERLEAVED ? 1 : p.pairs;           // from a pair's first vector to its second
    for (int j = threadIdx.x; j < p.pairs; j += kThreads) {
        const double f = p.turns[j];
        frequency[j] = f;
        split[j] = make_float2((float)f, (float)(f - (float)f));
        axis[j] = p.axis[j];
    }
    bool formed = false;
    for (int i = threadIdx.x; i - (int)threadIdx.x < all; i += kUnits * kThreads) {
        Raw v[kUnits], u[kOne ? 1 : kUnits];
        int at[kUnits], cs[kUnits];       // in out; in the table, or less than 0: nothing to turn
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const bool turns = unit < turning;
            const int c = !turns ? 2 * p.pairs + (unit - turning) * VEC : INTERLEAVED && !WIDE ? 2 * unit : unit * VEC;
            at[k] = i + k * kThreads < all ? (token * p.G + head) * p.D + c : -1;
            cs[k] = turns ? token * 2 * p.pairs + (kOne ? unit * VEC / 2 : unit * VEC) : -1;
            if (at[k] >= 0) {
                const T *from = x + token * p.xs[1] + head * p.xs[2] + c;
                v[k] = *reinterpret_cast<const Raw *>(from);
                if constexpr (!kOne) {
                    if (turns) u[k] = *reinterpret_cast<const Raw *>(from + other);
                }
            }
            token += p.tokens, head += p.heads, unit += p.step;
            if (unit >= units) unit -= units, ++head;
            if (head >= p.G) head -= p.G, ++token;
        }
        if (!formed) {
            __syncthreads();
            int of = over(threadIdx.x, p.pairs_inverse), pair = threadIdx.x - of * p.pairs;
            const int64_t from = b * p.ps[0] + first * p.ps[1];
            for (int j = threadIdx.x; j < count * p.pairs; j += kThreads) {
                const int64_t place = from + of * p.ps[1] + axis[pair] * p.ps[2];
                float turns, s, c;
                if (p.position_dtype == MSDA_B200_F32) {
                    const float at = __ldg(static_cast<const float *>(p.positions) + place), most = __fmul_rn(at, split[pair].x);
                    const float rest = __fmaf_rn(at, split[pair].y, __fmaf_rn(at, split[pair].x, -most));
                    turns = (most - nearest(most)) + rest;
                    turns -= nearest(turns);
                    if (!(fabsf(most) < kFarTurns)) turns = far_turns(at, frequency[pair]);
                } else {
                    turns = far_turns(position(p, place), frequency[pair]);
                }
                sine_cosine<T>(turns, s, c);
                table[of * 2 * p.pairs + pair] = c;
                table[of * 2 * p.pairs + p.pairs + pair] = s * p.sign;
                of += p.pair_tokens, pair += p.pair_step;
                if (pair >= p.pairs) pair -= p.pairs, ++of;
            }
            __syncthreads();
            formed = true;
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            if (at[k] < 0) continue;
            if (cs[k] >= 0) {
                const float *c = table + cs[k], *s = c + p.pairs;
                if constexpr (!WIDE) {
                    float y = VecTraits<T>::to_float(v[k]), z = VecTraits<T>::to_float(u[k]);
                    turn(y, z, *c, *s);
                    v[k] = VecTraits<T>::from_float(y);
                    out[at[k] + other] = VecTraits<T>::from_float(z);
                } else if constexpr (INTERLEAVED) {
                    float2 y[VEC / 2];
                    VecTraits<T>::unpack(v[k], y);
#pragma unroll
                    for (int j = 0; j < VEC / 2; j += 2) {
                        const float2 c2 = *reinterpret_cast<const float2 *>(c + j), s2 = *reinterpret_cast<const float2 *>(s + j);
                        turn(y[j].x, y[j].y, c2.x, s2.x);
                        turn(y[j + 1].x, y[j + 1].y, c2.y, s2.y);
                    }
                    v[k] = VecTraits<T>::pack(y);
                } else {
                    float2 y[VEC / 2], z[VEC / 2];
                    VecTraits<T>::unpack(v[k], y);
                    VecTraits<T>::unpack(u[k], z);
#pragma unroll
                    for (int j = 0; j < VEC / 2; j += 2) {
                        const float4 c4 = *reinterpret_cast<const float4 *>(c + 2 * j), s4 = *reinterpret_cast<const float4 *>(s + 2 * j);
                        turn2(y[j], z[j], make_float2(c4.x, c4.y), make_float2(s4.x, s4.y));
                        turn2(y[j + 1], z[j + 1], make_float2(c4.z, c4.w), make_float2(s4.z, s4.w));
                    }
                    v[k] = VecTraits<T>::pack(y);
                    *reinterpret_cast<uint4 *>(out + at[k] + other) = VecTraits<T>::pack(z);
                }
            }
            *reinterpret_cast<Raw *>(out + at[k]) = v[k];
        }
    }
}

template <typename T, bool WIDE, bool INTERLEAVED>
cudaError_t launch(RotaryParams p, unsigned grid, cudaStream_t stream) {
    constexpr int VEC = WIDE ? 16 / sizeof(T) : 1;
    p.turning = (INTERLEAVED && WIDE ? 2 : 1) * p.pairs / VEC;
    p.units = p.turning + (p.D - 2 * p.pairs) / VEC;
    p.per_token = p.G * p.units;
    p.tokens = kThreads / p.per_token, p.heads = kThreads % p.per_token / p.units, p.step = kThreads % p.per_token % p.units;
    const int pairs = std::max(p.pairs, 1);
    p.pair_tokens = kThreads / pairs, p.pair_step = kThreads % pairs;
    p.per_token_inverse = 1.f / p.per_token, p.units_inverse = 1.f / p.units, p.pairs_inverse = 1.f / pairs;
    rotary_kernel<T, WIDE, INTERLEAVED><<<grid, kThreads, p.tile * p.pairs * 2 * sizeof(float), stream>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const RotaryParams &p, bool interleaved, unsigned grid, cudaStream_t stream) {
    // 16-byte vectors where every one of them is aligned and belongs to one kind of unit
    constexpr int kVec = 16 / sizeof(T);
    const bool wide = p.D % kVec == 0 && (interleaved ? 2 * p.pairs : p.pairs) % kVec == 0 && p.xs[0] % kVec == 0 &&
                      p.xs[1] % kVec == 0 && p.xs[2] % kVec == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    if (interleaved) return wide ? launch<T, true, true>(p, grid, stream) : launch<T, false, true>(p, grid, stream);
    return wide ? launch<T, true, false>(p, grid, stream) : launch<T, false, false>(p, grid, stream);
}

int refuse(int status, const char *message) { return set_last_error(status, message); }

}  // namespace

}  // namespace msda_b200

extern "C" int msda_b200_rotary(const void *x, const int64_t *x_strides, const void *positions,
                                const int64_t *position_strides, int position_dtype, void *out, int64_t B, int64_t N,
                                int64_t G, int64_t D, int64_t axes, int64_t pairs, const double *frequencies,
                                const int *axis_of_pair, int interleaved, int inverse, int dtype, int device,
                                void *stream) {
    using namespace msda_b200;
    if (B < 0 || N < 0 || G <= 0 || D <= 0 || axes <= 0 || pairs < 0 || 2 * pairs > D || G > 1 << 20 || D > 1 << 20 ||
        N > 0x7fffffff || B > 0x7fffffff || G * D > 1 << 24)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: sizes out of range");
    if (pairs > kMostPairs) return refuse(MSDA_B200_UNSUPPORTED, "rotary: more than 128 pairs");
    if (dtype != MSDA_B200_F32 && dtype != MSDA_B200_F16 && dtype != MSDA_B200_BF16)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: dtype is not f32, f16 or bf16");
    if (position_dtype != MSDA_B200_F32 && position_dtype != MSDA_B200_F64 && position_dtype != MSDA_B200_I32 &&
        position_dtype != MSDA_B200_I64)
        return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: positions are not f32, f64, i32 or i64");
    if (B == 0 || N == 0) return MSDA_B200_OK;
    if (x == nullptr || x_strides == nullptr || positions == nullptr || position_strides == nullptr || out == nullptr ||
        (pairs > 0 && (frequencies == nullptr || axis_of_pair == nullptr)))
        return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: null pointer argument");
    RotaryParams p{};
    p.x = x, p.positions = positions, p.out = out;
    for (int i = 0; i < 3; ++i) p.xs[i] = x_strides[i], p.ps[i] = position_strides[i];
    p.N = (int)N, p.G = (int)G, p.D = (int)D, p.pairs = (int)pairs;
    p.position_dtype = position_dtype;
    p.sign = inverse ? -1.f : 1.f;
    for (int i = 0; i < pairs; ++i) {
        if (axis_of_pair[i] < 0 || axis_of_pair[i] >= axes || axis_of_pair[i] > 255)
            return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: a pair's axis is out of range");
        p.turns[i] = frequencies[i] * 0.15915494309189535;      // 1 / (2 pi)
        p.axis[i] = (uint8_t)axis_of_pair[i];
    }
    // As many tokens to a CTA as its threads ask for at a time, of 1 KB and more twice that, as long as every SM gets some;
    // the table within 32 KB.  Twice: 16 heads of 128 in float16 44.3 us in place of 47.8, 8 of 32 in float32 13.5 and
    // 13.7, but in bf16 (512 bytes, where it makes a table of 512 entries in a row) 18.8 and 17.5.
    const int64_t bytes = G * D * (dtype == MSDA_B200_F32 ? 4 : 2);
    int64_t tile = std::max<int64_t>(1, (bytes >= 1024 ? 4 : 2) * kInFlight * kThreads * 16 / bytes);
    tile = std::min(tile, std::max<int64_t>(1, B * N / (148 * 4)));
    if (pairs > 0) tile = std::min<int64_t>(tile, 4096 / pairs);
    tile = std::max<int64_t>(1, std::min(tile, N));
    p.tile = (int)tile;
    p.tiles = (unsigned)((N + tile - 1) / tile);
    const int64_t grid = B * ((N + tile - 1) / tile);
    if (grid > 0x7fffffff) return refuse(MSDA_B200_UNSUPPORTED, "rotary: too many tokens");
    const DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return refuse(MSDA_B200_CUDA_ERROR, cudaGetErrorString(guard.err));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == MSDA_B200_F32 ? launch_typed<float>(p, interleaved != 0, (unsigned)grid, s)
                          : dtype == MSDA_B200_F16 ? launch_typed<__half>(p, interleaved != 0, (unsigned)grid, s)
                                                   : launch_typed<__nv_bfloat16>(p, interleaved != 0, (unsigned)grid, s);
    if (e != cudaSuccess) return refuse(MSDA_B200_CUDA_ERROR, cudaGetErrorString(e));
    count_launches(1, 0);
    return MSDA_B200_OK;
}
