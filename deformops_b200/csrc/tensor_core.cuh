// Blackwell's asynchronous units as the attention kernels use them: mbarriers, tiled TMA loads,
// tcgen05 matrix instructions and tensor memory.  One CTA, no clusters.
//
// Operand tiles in shared memory are rows of 64 or 128 bytes, swizzled: the 16-byte chunk c of row r lies
// at r * pitch + 16 * (c ^ x), x = r % 8 (128-byte rows) or (r / 2) % 4 (64-byte rows).  Heads of 128
// channels are two such blocks of 64 channels behind one another.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

namespace msda_b200 {
namespace tc {

__device__ __forceinline__ uint32_t smem_address(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// one thread of the (whole) warp
__device__ __forceinline__ bool elect_one() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}

// ---- mbarriers ------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t at, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(at), "r"(parity)
                 : "memory");
    return done != 0;
}
// Whether the phase of this parity ended.  Bounded: a wait of 2^33 cycles (four seconds and more; no call gets
// there) lets its role leave, so that a mistake cannot hold the GPU.  A phase that is over costs 48 cycles so;
// a bounded loop from the first try on costs 170.
__device__ __forceinline__ bool barrier_wait(uint64_t *bar, uint32_t parity) {
    const uint32_t at = smem_address(bar);
    if (barrier_try(at, parity) || barrier_try(at, parity) || barrier_try(at, parity)) return true;
    uint32_t done;
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .u64 begun, now;\n\tmov.u64 begun, %%clock64;\n\t"
                 "again_%=:\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "@p bra over_%=;\n\t"
                 "mov.u64 now, %%clock64;\n\t"
                 "sub.u64 now, now, begun;\n\t"
                 "setp.lt.u64 q, now, %3;\n\t"
                 "@q bra again_%=;\n\t"
                 "over_%=:\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(at), "r"(parity), "n"(1ll << 33)
                 : "memory");
    return done != 0;
}

// Where one walks in a ring of SIZE barriers, and the parity of its round there.  Whoever waits for places to be free
// waits for the other parity: before the first round that is over.
template <int SIZE>
struct Ring {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next(int steps = 1) {
        at += steps;
        if (at >= SIZE) at -= SIZE, parity ^= 1;
    }
};

// plain stores to shared memory, before the asynchronous units read them (of barriers that were just made too: loads and
// products arrive on them)
__device__ __forceinline__ void fence_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- TMA ------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load(void *to, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_address(to)), "l"(map), "r"(smem_address(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}

// ---- tensor memory --------------------------------------------------------------------------------
// One whole warp.  Only then may the kernel behind this one begin (grid_launch_dependents): a CTA has said so as soon as one
// of its threads has, and a CTA of that kernel which took these columns first would hold them until this kernel ends,
// which could not end without them.
__device__ __forceinline__ void tmem_alloc(uint32_t *to, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(to)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {         // one whole warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the thread's own lane
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t (&r)[16], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t (&r)[8], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// loaded registers may be used from here on (the compiler has to be told: nothing else ties them to the wait)
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), 
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), 
                   "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void loaded(uint32_t (&r)[16]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), 
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void loaded(uint32_t (&r)[8]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- matrix instructions ---------------------------------------------------------------------------
// A shared memory descriptor has the address and the two strides (all in 16 bytes), version 1 and the swizzle of
// 128 or 64 bytes.  Rows along the product's k ("k-major"): STRIDE is that of eight rows, LEADING is not used.  Rows
// along the other axis: STRIDE is that of eight rows (of k), LEADING that of the next 64 (32) elements.  The upper
// half is a constant; offsets within a tile are added to the lower one.
template <int ROW_BYTES>
constexpr uint32_t kDescriptorHigh = (8 * ROW_BYTES >> 4) | 1u << 14 | (ROW_BYTES == 128 ? 2u : 4u) << 29;
__device__ __forceinline__ uint32_t descriptor(uint32_t at, uint32_t leading) { return at >> 4 | leading >> 4 << 16; }
// float32 sums of two 16-bit types alike; b_rows: B's rows run along k
__host__ __device__ constexpr uint32_t instruction(bool bf16, int m, int n, bool b_rows) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_rows ? 1u << 16 : 0u) |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// Issued by one thread, which has to be one that elect_one() chose: then the compiler knows that there is one,
// and every operand is in uniform registers (an `if (lane == 0)` costs about 100 cycles a product).
template <int ROW_BYTES>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
                 "r"((uint32_t)add), "n"(kDescriptorHigh<ROW_BYTES>)
                 : "memory");
}
// A from tensor memory: two 16-bit elements of k to a column
template <int ROW_BYTES>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
                 "r"((uint32_t)add), "n"(kDescriptorHigh<ROW_BYTES>)
                 : "memory");
}
// arrives on the barrier when everything that this thread has issued is done
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar))
                 : "memory");
}

// ---- swizzled tiles ---------------------------------------------------------------------------------
template <int DP>
constexpr int kRowBytes = DP == 32 ? 64 : 128;
// byte offset of the 16-byte chunk (of eight channels) `chunk` of `row`, in a tile of ROWS rows
template <int DP, int ROWS>
__device__ __forceinline__ int swizzled(int row, int chunk) {
    if constexpr (DP == 32) return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    const int block = chunk >> 3;
    return block * ROWS * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// ---- tensor maps -------------------------------------------------------------------------------------
// A (sample, token, head, D) tensor in tiles of rows.  Without shared heads a row is a token of one head;
// else the rows of a key head are its `share` query heads, token after token, and a tile has whole tokens.
struct TensorMap {
    CUtensorMap map;
    int axis_token, axis_head, axis_batch;       // 1 .. 3
    int share, one_batch, one_head;              // one_*: the same for all
};

// rows first .. of key head h; `first` is a multiple of share.  The barrier expects the bytes already.
template <int DP, int ROWS>
__device__ __forceinline__ void load_rows(unsigned char *to, const TensorMap &m, uint64_t *bar, int b, int h, int first) {
    const int token = m.share == 1 ? first : first / m.share;
    int c[4];
#pragma unroll
    for (int i = 1; i < 4; ++i)
        c[i] = i == m.axis_token ? token : i == m.axis_head ? (m.one_head ? 0 : h * m.share) : (m.one_batch ? 0 : b);
#pragma unroll
    for (int d = 0; d < DP; d += 64) tma_load(to + d * ROWS * 2, &m.map, bar, d, c[1], c[2], c[3]);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// the driver's function, asked for once
inline EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

// `heads` key heads of `share` heads each; false where TMA cannot describe the tensor so
template <typename T, int DP>
bool make_map(TensorMap &m, const void *base, const int64_t (&strides)[3], int B, int tokens, int heads, int share, int D,
              int tile_rows) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr || share > tile_rows) return false;
    struct Axis {
        int64_t stride, size;
        int what;
    } axes[3] = {{strides[0], B, 0}, {strides[1], tokens, 1}, {strides[2], (int64_t)heads * share, 2}};
    if ((strides[1] == 0 && tokens > 1) || (strides[2] == 0 && share > 1)) return false;
    m.share = share;
    m.one_batch = strides[0] == 0, m.one_head = strides[2] == 0;
    for (Axis &a : axes)
        if (a.stride == 0) a.size = 1;
    // axes from the densest on, but a tile's heads before its tokens; those of one element get a stride that fits
    const auto rank = [&](const Axis &a) { return a.stride == 0 ? INT64_MAX : a.stride; };
    std::stable_sort(axes, axes + 3, [&](const Axis &x, const Axis &y) { return rank(x) < rank(y); });
    if (share > 1) std::stable_sort(axes, axes + 3, [](const Axis &x, const Axis &y) { return x.what == 2 && y.what != 2; });
    cuuint64_t dims[4] = {(cuuint64_t)D, 0, 0, 0}, bytes[3];
    cuuint32_t box[4] = {(cuuint32_t)std::min(DP, 64), 1, 1, 1}, ones[4] = {1, 1, 1, 1};
    int64_t widest = (D + 7) / 8 * 8;
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = (cuuint64_t)axes[i].size;
        const int64_t stride = axes[i].stride != 0 ? axes[i].stride : widest;
        widest = std::max(widest, stride * axes[i].size);
        bytes[i] = (cuuint64_t)stride * 2;
        (axes[i].what == 0 ? m.axis_batch : axes[i].what == 1 ? m.axis_token : m.axis_head) = i + 1;
        if (axes[i].what == 1) box[i + 1] = (cuuint32_t)(tile_rows / share);
        if (axes[i].what == 2) box[i + 1] = (cuuint32_t)share;
    }
    return encode(&m.map, std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                  const_cast<void *>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  DP == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// Whether a block has the registers that its warps share out among them: they are those that the compiler gave it at
// launch, and an increase beyond them would wait for good.  Asked once for each kernel.
template <typename Kernel>
bool registers_suffice(Kernel kernel, int threads, int shared_out) {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && a.numRegs * threads >= shared_out;
}

}  // namespace tc
}  // namespace msda_b200
