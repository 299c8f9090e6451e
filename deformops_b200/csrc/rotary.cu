// Rotary positions of several axes: pairs of channels turned by position * frequency.
//
//   (a, b) -> (a cos - b sin, a sin + b cos),   angle = position of the pair's axis * its frequency
//
// One pass over x.  A CTA takes a few tokens: first it forms the sine and cosine of every (token, pair),
// once for all heads, then its threads turn 16-byte vectors of both halves of the pairs.  Angles
// are formed in 64 bits as turns and reduced to [-1/2, 1/2] before anything is rounded to 32: at
// position 10^6 a 32-bit angle is 0.03 off.  (float64 multiplies run at half the float32 rate here and
// there is one for each of G * D / pairs channels.)  The backward pass is the same kernel with the
// angles' sign turned.
#include <algorithm>

#include "../../include/msda_b200.h"
#include "msda_common.cuh"

namespace msda_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 128;

struct RotaryParams {
    const void *x, *positions;
    void *out;
    int64_t xs[3], ps[3];                 // strides of (sample, token, head), (sample, token, axis)
    int64_t tokens;                       // of all samples
    int N, G, D, pairs, tile;             // tile: tokens of a CTA
    int position_dtype;
    float sign;
    double turns[kMostPairs];             // frequency / 2 pi
    uint8_t axis[kMostPairs];
};

__device__ __forceinline__ double position(const RotaryParams &p, int64_t at) {
    switch (p.position_dtype) {
        case MSDA_B200_F32: return __ldg(static_cast<const float *>(p.positions) + at);
        case MSDA_B200_F64: return __ldg(static_cast<const double *>(p.positions) + at);
        case MSDA_B200_I32: return __ldg(static_cast<const int *>(p.positions) + at);
        default: return (double)__ldg(static_cast<const long long *>(p.positions) + at);
    }
}

template <typename T>
__device__ __forceinline__ void turn(T &x, T &y, float2 w) {
    const float a = VecTraits<T>::to_float(x), b = VecTraits<T>::to_float(y);
    // (written out, so that every variant of the kernel gives the same bits)
    x = VecTraits<T>::from_float(__fmaf_rn(a, w.x, __fmul_rn(-b, w.y)));
    y = VecTraits<T>::from_float(__fmaf_rn(a, w.y, __fmul_rn(b, w.x)));
}

// VEC elements to a load, 16 bytes or one element; INTERLEAVED: a pair is two neighbours, else the
// channels i and i + pairs
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    struct alignas(sizeof(T) * VEC) Vec {
        T v[VEC];
    };
    extern __shared__ float2 table[];     // (tile, pairs) of (cos, sin)
    const int64_t first = (int64_t)blockIdx.x * p.tile;
    const int count = (int)min((int64_t)p.tile, p.tokens - first);
    for (int i = threadIdx.x; i < count * p.pairs; i += kThreads) {
        const int token = i / p.pairs, pair = i - token * p.pairs;
        const int64_t b = (first + token) / p.N, n = first + token - b * p.N;
        double turns = position(p, b * p.ps[0] + n * p.ps[1] + p.axis[pair] * p.ps[2]) * p.turns[pair];
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        table[i] = make_float2(c, s * p.sign);
    }
    __syncthreads();

    // a unit: two vectors of pairs (one of interleaved pairs where VEC > 1), or one behind the turned channels
    constexpr bool kOne = INTERLEAVED && VEC > 1;
    const int turning = (kOne ? 2 : 1) * p.pairs / VEC;
    const int units = turning + (p.D - 2 * p.pairs) / VEC;
    const int per_token = p.G * units;
    for (int i = threadIdx.x; i < count * per_token; i += kThreads) {
        const int token = i / per_token, rest = i - token * per_token, head = rest / units, unit = rest - head * units;
        const int64_t b = (first + token) / p.N, n = first + token - b * p.N;
        const T *x = static_cast<const T *>(p.x) + b * p.xs[0] + n * p.xs[1] + head * p.xs[2];
        T *out = static_cast<T *>(p.out) + ((first + token) * p.G + head) * p.D;
        const float2 *cs = table + token * p.pairs;
        if (unit >= turning) {
            const int c = 2 * p.pairs + (unit - turning) * VEC;
            *reinterpret_cast<Vec *>(out + c) = *reinterpret_cast<const Vec *>(x + c);
        } else if constexpr (kOne) {
            Vec v = *reinterpret_cast<const Vec *>(x + unit * VEC);
#pragma unroll
            for (int j = 0; j < VEC; j += 2) turn(v.v[j], v.v[j + 1], cs[(unit * VEC + j) / 2]);
            *reinterpret_cast<Vec *>(out + unit * VEC) = v;
        } else {
            const int c0 = INTERLEAVED ? 2 * unit : unit * VEC, c1 = INTERLEAVED ? 2 * unit + 1 : p.pairs + unit * VEC;
            Vec v = *reinterpret_cast<const Vec *>(x + c0), u = *reinterpret_cast<const Vec *>(x + c1);
#pragma unroll
            for (int j = 0; j < VEC; ++j) turn(v.v[j], u.v[j], cs[unit * VEC + j]);
            *reinterpret_cast<Vec *>(out + c0) = v;
            *reinterpret_cast<Vec *>(out + c1) = u;
        }
    }
}

template <typename T, int VEC, bool INTERLEAVED>
cudaError_t launch(const RotaryParams &p, cudaStream_t stream) {
    const int64_t grid = (p.tokens + p.tile - 1) / p.tile;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    rotary_kernel<T, VEC, INTERLEAVED><<<(unsigned)grid, kThreads, p.tile * p.pairs * sizeof(float2), stream>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const RotaryParams &p, bool interleaved, cudaStream_t stream) {
    // 16-byte vectors where every one of them is aligned and belongs to one kind of unit
    constexpr int kVec = 16 / sizeof(T);
    const bool wide = p.D % kVec == 0 && (interleaved ? 2 * p.pairs : p.pairs) % kVec == 0 && p.xs[0] % kVec == 0 &&
                      p.xs[1] % kVec == 0 && p.xs[2] % kVec == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    if (interleaved) return wide ? launch<T, kVec, true>(p, stream) : launch<T, 1, true>(p, stream);
    return wide ? launch<T, kVec, false>(p, stream) : launch<T, 1, false>(p, stream);
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
    p.tokens = B * N, p.N = (int)N, p.G = (int)G, p.D = (int)D, p.pairs = (int)pairs;
    p.position_dtype = position_dtype;
    p.sign = inverse ? -1.f : 1.f;
    for (int i = 0; i < pairs; ++i) {
        if (axis_of_pair[i] < 0 || axis_of_pair[i] >= axes || axis_of_pair[i] > 255)
            return refuse(MSDA_B200_INVALID_ARGUMENT, "rotary: a pair's axis is out of range");
        p.turns[i] = frequencies[i] * 0.15915494309189535;      // 1 / (2 pi)
        p.axis[i] = (uint8_t)axis_of_pair[i];
    }
    // about four vectors to a thread, as long as every SM gets some tokens; the table within 32 KB
    const int64_t bytes = G * D * (dtype == MSDA_B200_F32 ? 4 : 2);
    int64_t tile = std::max<int64_t>(1, 4 * kThreads * 16 / std::max<int64_t>(bytes, 1));
    tile = std::min(tile, std::max<int64_t>(1, p.tokens / (148 * 4)));
    if (pairs > 0) tile = std::min<int64_t>(tile, 4096 / pairs);
    p.tile = (int)std::max<int64_t>(1, tile);
    const DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return refuse(MSDA_B200_CUDA_ERROR, cudaGetErrorString(guard.err));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == MSDA_B200_F32 ? launch_typed<float>(p, interleaved != 0, s)
                          : dtype == MSDA_B200_F16 ? launch_typed<__half>(p, interleaved != 0, s)
                                                   : launch_typed<__nv_bfloat16>(p, interleaved != 0, s);
    if (e != cudaSuccess) return refuse(MSDA_B200_CUDA_ERROR, cudaGetErrorString(e));
    count_launches(1, 0);
    return MSDA_B200_OK;
}
