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
        const int page = __ldg(table + b * stride + p);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(count)) return -1;
        return page * size + (slot - static_cast<int>(p) * size);
    }
    // Slots in use, cut to what the table can name.
    __device__ __forceinline__ int length(const int* lengths, int b, int* status, bool tell) const {
        const int n = __ldg(lengths + b), most = per_seq * size;
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

// Eight consecutive elements of a 16-bit or 32-bit type, as FP32.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Eight<__half> {
    uint4 v;
    __device__ __forceinline__ void load(const __half* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
    static __device__ __forceinline__ void store(__half* p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
};

}  // namespace serve
