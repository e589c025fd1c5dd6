// Head norms with the position rotation, forward and backward, and the append to a gather cache, which is the same
// pass with its results going to pages.
//
// For a head row x of D elements, a learned scale w and the rotation Rot of the row's position,
//
//     y = Rot(w o x r),                 r = 1 / sqrt(mean(x^2) + eps)
//     g = Rot^T dy,   dw = sum_rows g o x r,   dx = r (w o g) - x r^3 mean(x o w o g).
//
// Rot turns pairs of the first `rot` columns by the angles whose cosines and sines a table holds: columns (d, d + rot/2),
// or neighbours (2d, 2d + 1).  A tensor without w is rotated only, one without `rotate` normed only; the cache's value
// rows are neither.
//
// Both directions are bound by memory traffic: a row is read once and written once, everything between stays in
// registers.  D / 8 neighbouring lanes hold a row (16 bytes a lane and 16-bit element), so the mean is a few shuffles
// and the rotation's partner one shuffle away.  Such a group takes up to four heads of one token: four loads in
// flight a lane, and the token's angles are fetched once for them.  All of a call's tensors go in one launch, each
// with its own range of blocks.  The backward keeps the columns of dw that a lane owns in registers over all rows
// that it visits; blocks write their sums to a plane each, which a second kernel adds in a fixed order, so that
// repeated calls agree to the bit.
#include <algorithm>

#include "att3_abi_internal.h"
#include "serve_common.cuh"

namespace {

using serve::Eight;

__device__ int g_serve_status = 0;

constexpr int THREADS = 256;
constexpr int HEADS_PER_ITEM = 4;
constexpr int MAX_TENSORS = 5;
constexpr int BWD_BLOCKS_PER_SM = 4;

enum RotMode { ROT_NONE = 0, ROT_LANES = 1, ROT_IN_LANE = 2, ROT_NEIGHBOURS = 3 };

struct Tensor {
    const void* x;
    void* y;
    const void* dy;
    void* dx;
    const void* w;
    float* dw;
    long long xs[3], ys[3], dys[3], dxs[3];
    int w_type, rotate, heads, items, block0, blocks;      // items: groups of up to four heads in a token
};

struct Params {
    Tensor t[MAX_TENSORS];
    int n;
    const float* table;
    const void* positions;
    long long pos_b, pos_n;
    int pos_bytes, table_rows, rot, mode;
    int B, N;
    float eps;
    float* partial;                                // backward: [blocks][D]
    // append
    serve::Pages pages;
    const int* lengths;
    const int* counts;
    float* mass;
    int Hkv;
    int* status;
};

__device__ __forceinline__ void load_scale(const Tensor& t, int col, float (&w)[8]) {
    if (t.w_type == 0) { Eight<__nv_bfloat16> v; v.load(static_cast<const __nv_bfloat16*>(t.w) + col); v.get(w); }
    else if (t.w_type == 1) { Eight<__half> v; v.load(static_cast<const __half*>(t.w) + col); v.get(w); }
    else { Eight<float> v; v.load(static_cast<const float*>(t.w) + col); v.get(w); }
}

// A lane's eight cosines and signed sines: y'[k] = y[k] c[k] + partner[k] s[k].
__device__ __forceinline__ void load_angles(const Params& p, int pos, int lane_in_row, float (&c)[8], float (&s)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) { c[k] = 1.f; s[k] = 0.f; }
    if (p.mode == ROT_NONE || lane_in_row * 8 >= p.rot) return;
    const int half = p.rot >> 1;
    const float* row = p.table + static_cast<long long>(pos) * p.rot;
    if (p.mode == ROT_LANES) {
        const bool first = lane_in_row * 8 < half;
        const int at = lane_in_row * 8 - (first ? 0 : half);
        const float4 c0 = __ldg(reinterpret_cast<const float4*>(row + at)), c1 = __ldg(reinterpret_cast<const float4*>(row + at + 4));
        const float4 s0 = __ldg(reinterpret_cast<const float4*>(row + half + at)), s1 = __ldg(reinterpret_cast<const float4*>(row + half + at + 4));
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
        s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
        if (first) {
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] = -s[k];
        }
    } else {
        // four angles: of the pairs (k, k + 4) of the only rotated lane, or of the neighbours (2k, 2k + 1)
        const int at = p.mode == ROT_IN_LANE ? 0 : lane_in_row * 4;
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(row + at));
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(row + half + at));
        if (p.mode == ROT_IN_LANE) {
            c[0] = c[4] = c4.x; c[1] = c[5] = c4.y; c[2] = c[6] = c4.z; c[3] = c[7] = c4.w;
            s[4] = s4.x; s[5] = s4.y; s[6] = s4.z; s[7] = s4.w;
            s[0] = -s4.x; s[1] = -s4.y; s[2] = -s4.z; s[3] = -s4.w;
        } else {
            c[0] = c[1] = c4.x; c[2] = c[3] = c4.y; c[4] = c[5] = c4.z; c[6] = c[7] = c4.w;
            s[1] = s4.x; s[3] = s4.y; s[5] = s4.z; s[7] = s4.w;
            s[0] = -s4.x; s[2] = -s4.y; s[4] = -s4.z; s[6] = -s4.w;
        }
    }
}

// In place: y c + partner s (sign = 1), or the transposed rotation (sign = -1).  Every lane of the warp calls it.
template <int LANES>
__device__ __forceinline__ void rotate(int mode, int rot, int lane_in_row, float (&y)[8], const float (&c)[8],
                                       const float (&s)[8], float sign) {
    if (mode == ROT_NONE) return;
    float o[8];
    if (mode == ROT_LANES) {
        const int shift = rot >> 4;                                    // lanes in half of the rotated columns
        int from = lane_in_row < shift ? lane_in_row + shift : lane_in_row - shift;
        if (lane_in_row * 8 >= rot) from = lane_in_row;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = __shfl_sync(0xFFFFFFFFu, y[k], from, LANES);
    } else if (mode == ROT_IN_LANE) {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = y[k ^ 4];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = y[k ^ 1];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = y[k] * c[k] + sign * (o[k] * s[k]);
}

template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o >= 1; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o, LANES);
    return v;
}

__device__ __forceinline__ int find_tensor(const Params& p) {
    int ti = 0;
#pragma unroll
    for (int k = 1; k < MAX_TENSORS; ++k)
        if (k < p.n && static_cast<int>(blockIdx.x) >= p.t[k].block0) ti = k;
    return ti;
}

__device__ __forceinline__ int position_of(const Params& p, int b, int n) {
    long long pos = n;
    if (p.positions) {
        const long long at = b * p.pos_b + n * p.pos_n;
        pos = p.pos_bytes == 8 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
    }
    if (pos < 0 || pos >= p.table_rows) {
        if (p.mode != ROT_NONE) serve::report(p.status, serve::ST_POSITION);
        pos = 0;
    }
    return static_cast<int>(pos);
}

// One group of D / 8 lanes takes up to four heads of one token.  PAGED: the results of all tensors but the fifth (the
// queries) go to the cache rows of slot lengths[b] + n, and that slot is the position unless `positions` names the
// position of the first new token.
template <typename XT, int D, bool PAGED>
__global__ void __launch_bounds__(THREADS) norm_rotate_kernel(const __grid_constant__ Params p) {
    constexpr int LANES = D / 8;
    const int ti = find_tensor(p);
    const Tensor& t = p.t[ti];
    const int lr = threadIdx.x % LANES;
    const long long item = static_cast<long long>(blockIdx.x - t.block0) * (THREADS / LANES) + threadIdx.x / LANES;
    const long long tokens = static_cast<long long>(p.B) * p.N;
    const long long token = item / t.items;
    const int head0 = static_cast<int>(item - token * t.items) * HEADS_PER_ITEM;
    const bool live = token < tokens;
    const int b = live ? static_cast<int>(token / p.N) : 0, n = live ? static_cast<int>(token - static_cast<long long>(b) * p.N) : 0;

    Eight<XT> raw[HEADS_PER_ITEM];
    const XT* x = static_cast<const XT*>(t.x) + b * t.xs[0] + n * t.xs[1] + lr * 8;
#pragma unroll
    for (int u = 0; u < HEADS_PER_ITEM; ++u)
        if (live && head0 + u < t.heads) raw[u].load(x + (head0 + u) * t.xs[2]);

    long long dst = -1;                                                 // element offset of (row, head 0, column of this lane)
    int pos = 0;
    if (live) {
        if (PAGED) {
            const int slot = __ldg(p.lengths + b) + n;
            if (p.mode != ROT_NONE && t.rotate) {
                long long at = p.positions ? static_cast<long long>(static_cast<const int*>(p.positions)[b]) + n : slot;
                if (at < 0 || at >= p.table_rows) { serve::report(p.status, serve::ST_POSITION); at = 0; }
                pos = static_cast<int>(at);
            }
            if (ti < 4) {
                if (!p.counts || n < __ldg(p.counts + b)) {
                    const int row = p.pages.row(b, slot);
                    if (row < 0) serve::report(p.status, serve::ST_PAGE);
                    else dst = static_cast<long long>(row) * p.Hkv * D + lr * 8;
                    if (ti == 0 && p.mass && row >= 0 && lr == 0)
                        for (int u = 0; u < HEADS_PER_ITEM; ++u)
                            if (head0 + u < t.heads) p.mass[static_cast<long long>(row) * p.Hkv + head0 + u] = 0.f;
                }
            } else {
                dst = b * t.ys[0] + n * t.ys[1] + lr * 8;
            }
        } else {
            if (t.rotate) pos = position_of(p, b, n);
            dst = b * t.ys[0] + n * t.ys[1] + lr * 8;
        }
    }
    const long long step = PAGED && ti < 4 ? D : t.ys[2];
    float c[8], s[8], w[8];
    if (t.rotate) load_angles(p, pos, lr, c, s);
    if (t.w) load_scale(t, lr * 8, w);
#pragma unroll
    for (int u = 0; u < HEADS_PER_ITEM; ++u) {
        if (u >= t.heads) break;                                        // the same for the whole block
        float y[8];
        const bool here = live && head0 + u < t.heads;
        if (here) raw[u].get(y);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = 0.f;
        }
        if (t.w) {
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) ss += y[k] * y[k];
            const float r = 1.f / sqrtf(row_sum<LANES>(ss) * (1.f / D) + p.eps);
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = y[k] * r * w[k];
        }
        if (t.rotate) rotate<LANES>(p.mode, p.rot, lr, y, c, s, 1.f);
        if (here && dst >= 0) Eight<__nv_bfloat16>::store(static_cast<__nv_bfloat16*>(t.y) + dst + (head0 + u) * step, y);
    }
}

template <typename XT, int D>
__global__ void __launch_bounds__(THREADS) norm_rotate_backward_kernel(const __grid_constant__ Params p) {
    constexpr int LANES = D / 8, GROUPS = THREADS / LANES;
    __shared__ float sums[GROUPS][D];
    const int ti = find_tensor(p);
    const Tensor& t = p.t[ti];
    const int lr = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const long long tokens = static_cast<long long>(p.B) * p.N, items = tokens * t.items;
    float w[8], dw[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) { w[k] = 1.f; dw[k] = 0.f; }
    if (t.w) load_scale(t, lr * 8, w);

    // every lane of a warp makes the same number of turns: the shuffles want all of them
    for (long long base = static_cast<long long>(blockIdx.x - t.block0) * GROUPS; base < items;
         base += static_cast<long long>(t.blocks) * GROUPS) {
        const long long item = base + group;
        const bool live = item < items;
        const long long token = live ? item / t.items : 0;
        const int head0 = live ? static_cast<int>(item - token * t.items) * HEADS_PER_ITEM : 0;
        const int b = static_cast<int>(token / p.N), n = static_cast<int>(token - static_cast<long long>(b) * p.N);
        const XT* x = static_cast<const XT*>(t.x) + b * t.xs[0] + n * t.xs[1] + lr * 8;
        const __nv_bfloat16* dy = static_cast<const __nv_bfloat16*>(t.dy) + b * t.dys[0] + n * t.dys[1] + lr * 8;
        XT* dx = static_cast<XT*>(t.dx) + b * t.dxs[0] + n * t.dxs[1] + lr * 8;
        Eight<XT> rx[HEADS_PER_ITEM];
        Eight<__nv_bfloat16> rg[HEADS_PER_ITEM];
#pragma unroll
        for (int u = 0; u < HEADS_PER_ITEM; ++u)
            if (live && head0 + u < t.heads) {
                rg[u].load(dy + (head0 + u) * t.dys[2]);
                if (t.w) rx[u].load(x + (head0 + u) * t.xs[2]);
            }
        float c[8], s[8];
        if (t.rotate) load_angles(p, live ? position_of(p, b, n) : 0, lr, c, s);
#pragma unroll
        for (int u = 0; u < HEADS_PER_ITEM; ++u) {
            if (u >= t.heads) break;
            const bool here = live && head0 + u < t.heads;
            float g[8], v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) g[k] = v[k] = 0.f;
            if (here) {
                rg[u].get(g);
                if (t.w) rx[u].get(v);
            }
            if (t.rotate) rotate<LANES>(p.mode, p.rot, lr, g, c, s, -1.f);
            if (t.w) {
                float ss = 0.f, m = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    ss += v[k] * v[k];
                    m += v[k] * (w[k] * g[k]);
                }
                ss = row_sum<LANES>(ss);
                m = row_sum<LANES>(m);
                const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
                const float f = r * r * (m * r) * (1.f / D);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    dw[k] += g[k] * (v[k] * r);
                    g[k] = r * (w[k] * g[k]) - v[k] * f;
                }
            }
            if (here) Eight<XT>::store(dx + (head0 + u) * t.dxs[2], g);
        }
    }
    if (!t.w) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[group][lr * 8 + k] = dw[k];
    __syncthreads();
    if (threadIdx.x < D) {
        float a = 0.f;
        for (int q = 0; q < GROUPS; ++q) a += sums[q][threadIdx.x];
        p.partial[static_cast<long long>(blockIdx.x) * D + threadIdx.x] = a;
    }
}

// dw of one tensor a block: the planes of its blocks, added in a fixed order (a strided quarter or more each, then those).
template <int D>
__global__ void __launch_bounds__(1024) scale_grad_kernel(const __grid_constant__ Params p) {
    constexpr int PARTS = 1024 / D;
    __shared__ float sums[PARTS][D];
    const Tensor& t = p.t[blockIdx.x];
    if (!t.w) return;
    const int col = threadIdx.x % D, part = threadIdx.x / D;
    float a = 0.f;
#pragma unroll 8
    for (int q = part; q < t.blocks; q += PARTS) a += p.partial[static_cast<long long>(t.block0 + q) * D + col];
    sums[part][col] = a;
    __syncthreads();
    if (part == 0) {
        for (int q = 1; q < PARTS; ++q) a += sums[q][col];
        t.dw[col] = a;
    }
}

size_t element(int type) { return type == 2 ? 4 : 2; }

bool aligned(const void* ptr, const int64_t* strides, int type) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return false;
    for (int k = 0; strides && k < 3; ++k)
        if (strides[k] * static_cast<int64_t>(element(type)) % 16 != 0) return false;
    return true;
}

// Checks and fills what forward, backward and append have in common.  Blocks of a tensor: one group per item, or
// (persistent) a share of `budget` blocks in proportion to its rows.
int fill(Params& p, const char* who, const att3_head_rows* t, int n, int x_type, const float* table, int table_rows,
         int rot, int interleaved, int B, int N, int D, float eps, int budget) {
    if (!t || n < 1 || n > MAX_TENSORS) return att3::set_error(ATT3_ERR_INVALID, "%s: 1 to %d tensors, got %d", who, MAX_TENSORS, n);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return att3::set_error(ATT3_ERR_INVALID, "%s: head dim must be 16, 32, 64 or 128, got %d", who, D);
    if (B < 0 || N < 0) return att3::set_error(ATT3_ERR_INVALID, "%s: negative batch or length", who);
    if (x_type < 0 || x_type > 2) return att3::set_error(ATT3_ERR_INVALID, "%s: unknown element type %d", who, x_type);
    if (!(eps >= 0.f)) return att3::set_error(ATT3_ERR_INVALID, "%s: eps must not be negative", who);
    if (rot < 0 || rot > D || (rot % 16 != 0 && rot != 8))
        return att3::set_error(ATT3_ERR_INVALID, "%s: rotated columns must be 0, 8 or a multiple of 16 up to the head dim %d, got %d", who, D, rot);
    if (rot && (!table || table_rows < 1 || reinterpret_cast<uintptr_t>(table) % 16 != 0))
        return att3::set_error(ATT3_ERR_INVALID, "%s: the rotation needs a 16-byte aligned table with at least one row", who);
    p.n = n;
    p.table = table;
    p.table_rows = table_rows;
    p.rot = rot;
    p.mode = rot == 0 ? ROT_NONE : interleaved ? ROT_NEIGHBOURS : rot == 8 ? ROT_IN_LANE : ROT_LANES;
    p.B = B;
    p.N = N;
    p.eps = eps;
    const long long groups = THREADS / (D / 8);
    long long rows = 0, blocks = 0;
    for (int k = 0; k < n; ++k) {
        if (t[k].heads < 1 || t[k].heads > (1 << 20)) return att3::set_error(ATT3_ERR_INVALID, "%s: tensor %d has no heads", who, k);
        rows += t[k].heads;
    }
    for (int k = 0; k < n; ++k) {
        Tensor& o = p.t[k];
        o.x = t[k].x; o.y = t[k].y; o.dy = t[k].dy; o.dx = t[k].dx; o.w = t[k].w; o.dw = t[k].dw;
        o.w_type = static_cast<int>(t[k].w_type);
        o.rotate = t[k].rotate != 0;
        for (int q = 0; q < 3; ++q) {
            o.xs[q] = t[k].x_stride[q]; o.ys[q] = t[k].y_stride[q]; o.dys[q] = t[k].dy_stride[q]; o.dxs[q] = t[k].dx_stride[q];
        }
        if (o.w && (o.w_type < 0 || o.w_type > 2)) return att3::set_error(ATT3_ERR_INVALID, "%s: unknown element type of scale %d", who, k);
        if (o.w && reinterpret_cast<uintptr_t>(o.w) % 16 != 0) return att3::set_error(ATT3_ERR_INVALID, "%s: scale %d must be 16-byte aligned", who, k);
        o.heads = static_cast<int>(t[k].heads);
        o.items = (o.heads + HEADS_PER_ITEM - 1) / HEADS_PER_ITEM;
        const long long items = static_cast<long long>(B) * N * o.items;
        long long nb = (items + groups - 1) / groups;
        if (budget) nb = std::min(nb, std::max<long long>(1, budget * static_cast<long long>(o.heads) / rows));
        o.block0 = static_cast<int>(blocks);
        o.blocks = static_cast<int>(nb);
        blocks += nb;
        if (blocks > 0x7FFFFFFFll) return att3::set_error(ATT3_ERR_INVALID, "%s: too many rows", who);
    }
    return ATT3_OK;
}

int total_blocks(const Params& p) { return p.t[p.n - 1].block0 + p.t[p.n - 1].blocks; }

template <bool PAGED>
int launch_forward(const Params& p, int x_type, int D, cudaStream_t st, const char* who) {
    const int blocks = total_blocks(p);
    if (blocks == 0) return ATT3_OK;
#define ATT3_NR(T, DD) norm_rotate_kernel<T, DD, PAGED><<<blocks, THREADS, 0, st>>>(p)
#define ATT3_NR_D(T) do { if (D == 16) ATT3_NR(T, 16); else if (D == 32) ATT3_NR(T, 32); else if (D == 64) ATT3_NR(T, 64); else ATT3_NR(T, 128); } while (0)
    if (x_type == 0) ATT3_NR_D(__nv_bfloat16);
    else if (x_type == 1) ATT3_NR_D(__half);
    else ATT3_NR_D(float);
#undef ATT3_NR_D
#undef ATT3_NR
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ATT3_OK : att3::set_cuda_error(e, who);
}

}  // namespace

namespace att3 {

// Device address of the serving kernels' status word on the current device (looked up once per device and thread).
int* serve_status_ptr() {
    constexpr int kMaxDevices = 64;
    static thread_local int* cached[kMaxDevices] = {nullptr};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
    if (!cached[dev]) {
        int* q = nullptr;
        if (cudaGetSymbolAddress(reinterpret_cast<void**>(&q), g_serve_status) != cudaSuccess) return nullptr;
        cached[dev] = q;
    }
    return cached[dev];
}

int serve_status_read_and_clear(int* out) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_serve_status, sizeof(int));
    if (e != cudaSuccess) return set_cuda_error(e, "att3_device_status: read");
    if (*out) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_serve_status, &zero, sizeof(int));
    }
    return ATT3_OK;
}

}  // namespace att3

extern "C" int att3_norm_rotate_forward(const att3_head_rows* tensors, int n, int x_type, const float* table, int table_rows,
                                        int rot, int interleaved, const void* positions, int pos_bytes, int64_t pos_b,
                                        int64_t pos_n, int B, int N, int D, float eps, void* stream) {
    const char* who = "att3_norm_rotate_forward";
    Params p = {};
    if (int rc = fill(p, who, tensors, n, x_type, table, table_rows, rot, interleaved, B, N, D, eps, 0)) return rc;
    if (positions && pos_bytes != 4 && pos_bytes != 8) return att3::set_error(ATT3_ERR_INVALID, "%s: positions are 4 or 8 bytes wide", who);
    if (B == 0 || N == 0) return ATT3_OK;
    for (int k = 0; k < n; ++k) {
        if (!tensors[k].x || !tensors[k].y) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor %d", who, k);
        if (!aligned(tensors[k].x, tensors[k].x_stride, x_type) || !aligned(tensors[k].y, tensors[k].y_stride, 0))
            return att3::set_error(ATT3_ERR_INVALID, "%s: rows of tensor %d must be 16-byte aligned", who, k);
    }
    if (!att3::require_sm100(who)) return ATT3_ERR_UNSUPPORTED;
    p.positions = positions; p.pos_bytes = pos_bytes; p.pos_b = pos_b; p.pos_n = pos_n;
    if (!(p.status = att3::serve_status_ptr())) return att3::set_error(ATT3_ERR_CUDA, "%s: status word not resolvable", who);
    return launch_forward<false>(p, x_type, D, static_cast<cudaStream_t>(stream), who);
}

extern "C" size_t att3_norm_rotate_workspace_bytes(int n, int D) {
    if (n < 1 || n > MAX_TENSORS || D < 1) return 0;
    // one plane a block: the budget, and at least one block a tensor
    return (static_cast<size_t>(att3::sm_count()) * BWD_BLOCKS_PER_SM + n) * D * sizeof(float);
}

extern "C" int att3_norm_rotate_backward(const att3_head_rows* tensors, int n, int x_type, const float* table, int table_rows,
                                         int rot, int interleaved, const void* positions, int pos_bytes, int64_t pos_b,
                                         int64_t pos_n, int B, int N, int D, float eps, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    const char* who = "att3_norm_rotate_backward";
    Params p = {};
    const int budget = att3::sm_count() * BWD_BLOCKS_PER_SM;
    if (int rc = fill(p, who, tensors, n, x_type, table, table_rows, rot, interleaved, B, N, D, eps, budget)) return rc;
    if (positions && pos_bytes != 4 && pos_bytes != 8) return att3::set_error(ATT3_ERR_INVALID, "%s: positions are 4 or 8 bytes wide", who);
    const bool rows = B > 0 && N > 0;
    bool scaled = false;
    for (int k = 0; k < n; ++k) {
        const att3_head_rows& t = tensors[k];
        if (t.w) scaled = true;
        if (t.w && !t.dw) return att3::set_error(ATT3_ERR_INVALID, "%s: tensor %d has a scale and no room for its gradient", who, k);
        if (!rows) continue;
        if (!t.dy || !t.dx || (t.w && !t.x)) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor %d", who, k);
        if ((t.w && !aligned(t.x, t.x_stride, x_type)) || !aligned(t.dy, t.dy_stride, 0) || !aligned(t.dx, t.dx_stride, x_type))
            return att3::set_error(ATT3_ERR_INVALID, "%s: rows of tensor %d must be 16-byte aligned", who, k);
    }
    if (!workspace || workspace_bytes < att3_norm_rotate_workspace_bytes(n, D))
        return att3::set_error(ATT3_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, att3_norm_rotate_workspace_bytes(n, D));
    if (!att3::require_sm100(who)) return ATT3_ERR_UNSUPPORTED;
    p.positions = positions; p.pos_bytes = pos_bytes; p.pos_b = pos_b; p.pos_n = pos_n;
    p.partial = static_cast<float*>(workspace);
    if (!(p.status = att3::serve_status_ptr())) return att3::set_error(ATT3_ERR_CUDA, "%s: status word not resolvable", who);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int blocks = total_blocks(p);
    if (blocks) {
#define ATT3_NR(T, DD) norm_rotate_backward_kernel<T, DD><<<blocks, THREADS, 0, st>>>(p)
#define ATT3_NR_D(T) do { if (D == 16) ATT3_NR(T, 16); else if (D == 32) ATT3_NR(T, 32); else if (D == 64) ATT3_NR(T, 64); else ATT3_NR(T, 128); } while (0)
        if (x_type == 0) ATT3_NR_D(__nv_bfloat16);
        else if (x_type == 1) ATT3_NR_D(__half);
        else ATT3_NR_D(float);
#undef ATT3_NR_D
#undef ATT3_NR
    }
    if (scaled) {                                   // with no rows at all this writes the gradient's zeros
        if (D == 16) scale_grad_kernel<16><<<n, 1024, 0, st>>>(p);
        else if (D == 32) scale_grad_kernel<32><<<n, 1024, 0, st>>>(p);
        else if (D == 64) scale_grad_kernel<64><<<n, 1024, 0, st>>>(p);
        else scale_grad_kernel<128><<<n, 1024, 0, st>>>(p);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ATT3_OK : att3::set_cuda_error(e, who);
}

extern "C" int att3_gather_cache_append(const att3_head_rows* tensors, int n, int x_type, const float* table, int table_rows,
                                        int rot, int interleaved, const int* positions, const att3_gather_pages* pages,
                                        const int* lengths, const int* counts, float* mass, int B, int T, int D, float eps,
                                        void* stream) {
    const char* who = "att3_gather_cache_append";
    Params p = {};
    if (n != 4 && n != 5) return att3::set_error(ATT3_ERR_INVALID, "%s: R, S, Vr, Vs and optionally Q, got %d tensors", who, n);
    if (int rc = fill(p, who, tensors, n, x_type, table, table_rows, rot, interleaved, B, T, D, eps, 0)) return rc;
    if (B == 0 || T == 0) return ATT3_OK;
    if (int rc = att3::check_gather_pages(pages, who)) return rc;
    if (!lengths) return att3::set_error(ATT3_ERR_INVALID, "%s: null lengths", who);
    for (int k = 0; k < n; ++k) {
        if (!tensors[k].x || !tensors[k].y) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor %d", who, k);
        if (!aligned(tensors[k].x, tensors[k].x_stride, x_type) || !aligned(tensors[k].y, k == 4 ? tensors[k].y_stride : nullptr, 0))
            return att3::set_error(ATT3_ERR_INVALID, "%s: rows of tensor %d must be 16-byte aligned", who, k);
        if (k < 4 && tensors[k].heads != tensors[0].heads) return att3::set_error(ATT3_ERR_INVALID, "%s: R, S, Vr, Vs must have the same heads", who);
    }
    if (!att3::require_sm100(who)) return ATT3_ERR_UNSUPPORTED;
    p.positions = positions;
    p.pages = serve::make_pages(pages->table, pages->table_stride, pages->per_sequence, pages->pages, pages->page_size);
    p.lengths = lengths;
    p.counts = counts;
    p.mass = mass;
    p.Hkv = static_cast<int>(tensors[0].heads);
    if (!(p.status = att3::serve_status_ptr())) return att3::set_error(ATT3_ERR_CUDA, "%s: status word not resolvable", who);
    return launch_forward<true>(p, x_type, D, static_cast<cudaStream_t>(stream), who);
}
