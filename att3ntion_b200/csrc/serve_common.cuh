// What the serving kernels (head norms with rotation, gather-cache append, single-token gather, eviction) share:
// the paged pools' addressing, element types, and the status word they report to.
//
// A page number, position or length that lies outside its table is never followed.  The kernel leaves the access
// out, records which of the three it was in the status word and goes on, so a bad table reads as an error of
// att3_device_status and not as a fault.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace serve {

// The serving kernels are short and follow one another, so each is launched to be set up while the kernel before it in
// the stream runs out (programmatic dependent launch), and waits for that kernel's end itself, before it touches memory.
// Every thread does: a kernel that ended without waiting could end before the one it depends on.  What they read may
// have been written while they were already being set up, so none of it goes through read-only loads (__ldg), which want
// memory that stays as it is for a kernel's whole life.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

enum Status { ST_WAIT = 1, ST_PAGE = 0x100, ST_POSITION = 0x200, ST_LENGTH = 0x400 };

__device__ __forceinline__ void report(int* status, int what) { atomicOr(status, what); }

// Pools are [pages, page_size, Hkv, D] contiguous; table[b * stride + p] is the page of slots p * page_size ...
struct Pages {
    const int* table;
    long long stride;
    int per_seq;      // entries of a sequence's row in the table
    int count;        // pages in the pool
    int size;         // slots in a page
    int shift;        // its logarithm, or -1 if it is no power of two
    // Row (page * page_size + slot in page) of `slot`, or -1 if the table has no valid page for it.
    __device__ __forceinline__ int row(int b, int slot) const {
        const unsigned p = shift >= 0 ? static_cast<unsigned>(slot) >> shift : static_cast<unsigned>(slot) / static_cast<unsigned>(size);
        if (slot < 0 || p >= static_cast<unsigned>(per_seq)) return -1;
        const int page = table[b * stride + p];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(count)) return -1;
        return page * size + (slot - static_cast<int>(p) * size);
    }
    // Slots in use, cut to what the table can name.
    __device__ __forceinline__ int length(const int* lengths, int b, int* status, bool tell) const {
        const int n = lengths[b], most = per_seq * size;
        if (n >= 0 && n <= most) return n;
        if (tell) report(status, ST_LENGTH);
        return n < 0 ? 0 : most;
    }
};

inline Pages make_pages(const int* table, long long stride, long long per_seq, long long count, long long size) {
    int shift = -1;
    for (int k = 0; k < 31; ++k)
        if (size == 1ll << k) shift = k;
    return Pages{table, stride, static_cast<int>(per_seq), static_cast<int>(count), static_cast<int>(size), shift};
}

// Division of numbers below 2^31 by a divisor known to the host: q = (high word of n * mul, plus n) >> shift
// (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divide {
    unsigned mul, shift;
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>((__umulhi(static_cast<unsigned>(n), mul) + static_cast<unsigned>(n)) >> shift);
    }
};
inline Divide make_divide(int by) {
    unsigned l = 0;
    while ((1ull << l) < static_cast<unsigned long long>(by)) ++l;
    return Divide{static_cast<unsigned>(((1ull << 32) * ((1ull << l) - by)) / by + 1), l};
}

// Four consecutive elements of a 16-bit or 32-bit type, as FP32.
template <typename T> struct Four {
    uint2 v;                                     // 16-bit types
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void get(float* f) const;
    static __device__ __forceinline__ void store(T* p, const float* f);
};
template <> __device__ __forceinline__ void Four<__nv_bfloat16>::get(float* f) const {
    f[0] = __uint_as_float(v.x << 16);
    f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16);
    f[3] = __uint_as_float(v.y & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void Four<__nv_bfloat16>::store(__nv_bfloat16* p, const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <> __device__ __forceinline__ void Four<__half>::get(float* f) const {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
template <> __device__ __forceinline__ void Four<__half>::store(__half* p, const float* f) {
    const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <> struct Four<float> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void get(float* f) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
    static __device__ __forceinline__ void store(float* p, const float* f) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
};

}  // namespace serve
