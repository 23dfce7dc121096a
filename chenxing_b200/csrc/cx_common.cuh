// Shared helpers for libcxkv: status/error reporting, element conversion,
// the device-side error flag word, small PTX wrappers (mbarrier, TMA,
// ldmatrix, mma) used by the sm_100a kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/cxkv.h"

namespace cx {

// ---- host-side error reporting -------------------------------------------
void set_error(const std::string& msg);
int fail(int code, const std::string& msg);
int cuda_fail(cudaError_t e, const char* what);

#define CX_CUDA_CHECK(call)                                   \
    do {                                                      \
        cudaError_t e_ = (call);                              \
        if (e_ != cudaSuccess) return cx::cuda_fail(e_, #call); \
    } while (0)

inline int check_launch(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, what);
    return CX_OK;
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

inline int elem_bytes(int32_t dt) {
    switch (dt) {
        case CX_F32: return 4;
        case CX_BF16: return 2;
        case CX_F16: return 2;
        default: return 0;
    }
}

constexpr int kBlockTok = 16;                               // tokens per block of the TMA kernels
constexpr unsigned long long kWaitLimitNs = 2000000000ull;  // 2 s per wait

int num_sms();  // SM count of the current device (cached per device)

// Limit of the decode / verify pipeline waits of later launches, ns
// (cx_set_wait_limit_ns).
unsigned long long wait_limit_ns();

static inline int check_pool(const cx_pool* p) {
    if (!p) return fail(CX_ERR_SHAPE, "pool is NULL");
    if (!p->k || !p->v) return fail(CX_ERR_SHAPE, "pool buffers are NULL");
    if (p->n_layers <= 0 || p->n_blocks <= 0 || p->block_size <= 0 || p->n_kv_heads <= 0 ||
        p->head_dim <= 0)
        return fail(CX_ERR_SHAPE, "pool sizes must be positive");
    if (elem_bytes(p->dtype) == 0) return fail(CX_ERR_DTYPE, "unknown pool dtype");
    return CX_OK;
}

// ---- device-side error flags ---------------------------------------------
// One word per translation unit (no relocatable device code); cx_device_error
// reads and clears them all.
static __device__ unsigned int g_dev_flags = 0;

// This translation unit's word on the current device; nullptr: none.
static unsigned int* dev_flags() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, g_dev_flags) == cudaSuccess ? static_cast<unsigned int*>(p)
                                                                : nullptr;
}

unsigned int* dev_flags_scored();   // of cxkv_scored.cu
unsigned int* dev_flags_tree();     // of cxkv_tree.cu
unsigned int* dev_flags_latent();   // of cxkv_latent.cu

__device__ __forceinline__ void raise_flag(unsigned int bit) {
    atomicOr(&g_dev_flags, bit);
}

// ---- element conversion ---------------------------------------------------
template <typename T> struct Conv;
template <> struct Conv<float> {
    __device__ __forceinline__ static float to_f(float x) { return x; }
    __device__ __forceinline__ static float from_f(float x) { return x; }
};
template <> struct Conv<__nv_bfloat16> {
    __device__ __forceinline__ static float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ __forceinline__ static __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Conv<__half> {
    __device__ __forceinline__ static float to_f(__half x) { return __half2float(x); }
    __device__ __forceinline__ static __half from_f(float x) { return __float2half_rn(x); }
};

// Element `i` of an array whose element type is known at run time only.
__device__ __forceinline__ void store_as(void* p, int32_t dtype, int64_t i, float x) {
    if (dtype == CX_F32)
        static_cast<float*>(p)[i] = x;
    else if (dtype == CX_BF16)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else
        static_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ float load_as(const void* p, int32_t dtype, int64_t i) {
    return dtype == CX_F32    ? static_cast<const float*>(p)[i]
           : dtype == CX_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                              : __half2float(static_cast<const __half*>(p)[i]);
}

// Elements `i`, `i + 1` (i even, the array 8-byte aligned) of such an array.
__device__ __forceinline__ void store2_as(void* p, int32_t dtype, int64_t i, float x, float y) {
    if (dtype == CX_F32)
        *reinterpret_cast<float2*>(static_cast<float*>(p) + i) = make_float2(x, y);
    else if (dtype == CX_BF16)
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p) + i) =
            __floats2bfloat162_rn(x, y);
    else
        *reinterpret_cast<__half2*>(static_cast<__half*>(p) + i) = __floats2half2_rn(x, y);
}

// ---- drafted trees (cx_tree) ------------------------------------------------
struct TreeMask {
    const uint32_t* masks;   // [rows][words]; NULL: chains
    const int32_t* depths;   // [rows]
    int64_t words;
};

// Bits [u0, u0 + 32) of a row of `words` mask words; bits outside it are 0.
__device__ __forceinline__ uint32_t mask_bits32(const uint32_t* row, int words, int u0) {
    const int w = u0 >> 5, sh = u0 & 31;      // (floor, also below 0)
    const uint32_t lo = w >= 0 && w < words ? __ldg(row + w) : 0u;
    const uint32_t hi = sh && w + 1 >= 0 && w + 1 < words ? __ldg(row + w + 1) : 0u;
    return __funnelshift_r(lo, hi, sh);
}

// Nodes [u0, u0 + 32) that query row `row` (node u_row of its sequence) sees: those
// of its mask up to itself.
__device__ __forceinline__ uint32_t tree_bits(const TreeMask& t, int64_t row, int u_row, int u0) {
    const uint32_t m = mask_bits32(t.masks + row * t.words, (int)t.words, u0);
    const int n = u_row + 1 - u0;
    return n >= 32 ? m : n <= 0 ? 0u : m & ((1u << n) - 1);
}

// Where drafted key u of the sequence with query rows [q0, q0 + n) stands: base + its depth.
__device__ __forceinline__ int tree_key_pos(const TreeMask& t, int64_t q0, int n, int base, int u) {
    return u >= 0 && u < n ? base + __ldg(t.depths + q0 + u) : base + u;
}

// Asynchronous 16-byte copy to shared memory; zeros when `there` is not set.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
                 "r"(there ? 16 : 0)
                 : "memory");
}

// ---- ends of a softmax ------------------------------------------------------
// A row's weight from its sum of exponentials: 0 where it saw no key.  NaN stays NaN (a
// comparison with `> 0` would turn a row of NaN scores into zeros).
__device__ __forceinline__ float sum_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }

// The reference that exponentials are taken against: 0 for a part whose scores have no
// maximum.  The weight of its sum is then 0 (2^-inf), and 0 * NaN hands on the NaN of scores
// that were no numbers.
__device__ __forceinline__ float ref_base(float m) { return m == -INFINITY ? 0.f : m; }

// ---- packed fp32 pairs ------------------------------------------------------
using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_of(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_get(f2 v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// ---- shared-memory / PTX helpers -----------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
                 : "memory");
}

__device__ __forceinline__ void fence_mbar_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
                 "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait on an mbarrier phase.  Gives up after `limit_ns` nanoseconds
// or as soon as *abort is set (abort may be NULL), and reports whether the
// phase completed.  Both are looked at after every EVERY-th try.  A try suspends
// the thread, and where few threads arrive 64 of them outlast long waits (some
// 70 us on the stages of the staged append): such waits look after each.
template <uint32_t EVERY = 64>
__device__ __forceinline__ bool mbar_wait_bounded(uint64_t* bar, uint32_t parity,
                                                  volatile int* abort, uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = global_ns();
    uint32_t spins = 0;
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((++spins & (EVERY - 1)) == 0) {
            if (abort && *abort) return false;
            if (global_ns() - t0 > limit_ns) return false;
        }
    }
}

// 3-D tiled TMA load into this CTA's own shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int x,
                                            int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

// 16-byte shared-memory store / load of four words.  The load is volatile so
// that it stays where it is written (inside a loop) instead of being hoisted
// into registers.
__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
}

__device__ __forceinline__ void ld_shared_v4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// D = A(16x16 bf16, row) * B(16x8 bf16, col) + D, fp32 accumulate.
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same on fp16 operands.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Two fp32 values as a 16-bit pair of type E, and the mma of that type.
template <typename E> struct Half16;
template <> struct Half16<__nv_bfloat16> {
    // A softmax reference (base 2) is set kLeadLog2 above its row's maximum and
    // follows when the maximum is kGrowLog2 above it: it then follows once in 60
    // powers of two, and no probability is above 2^8, so that their products with V
    // overflow no earlier than those of a reference that stays near the maximum.
    // (The price: a product with V below 2^-74 may fall below fp32's normal range.)
    static constexpr float kGrowLog2 = 8.f, kLeadLog2 = 52.f;
    static constexpr uint32_t kOnes = 0x3f803f80u;   // a pair of ones
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
    __device__ __forceinline__ static f2 unpack(uint32_t u) {
        return f2_of(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        mma_bf16_16816(d, a, b0, b1);
    }
};
template <> struct Half16<__half> {
    // fp16 holds 2^15 above the reference and loses bits 2^14 below it: no lead.
    static constexpr float kGrowLog2 = 15.f, kLeadLog2 = 0.f;
    static constexpr uint32_t kOnes = 0x3c003c00u;
    __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    __device__ __forceinline__ static f2 unpack(uint32_t u) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u));
        return f2_of(v.x, v.y);
    }
    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        mma_f16_16816(d, a, b0, b1);
    }
};

__device__ __forceinline__ void named_bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Arrive at named barrier `id` (of `threads` threads) without waiting.
__device__ __forceinline__ void named_bar_arrive(int id, int threads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

}  // namespace cx
