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
// registers.  D / 8 neighbouring lanes hold a row, eight columns a lane.  Which eight follows the rotation: four of the
// first half of the rotated columns and their four partners, or neighbours; so a lane turns its pairs by itself with
// four angles, and only the mean needs the row's other lanes.  (Eight neighbouring columns a lane, the partner's fetched
// by shuffles, took 394 instructions for two rows of 128 and 2.3 TB/s in the backward.)  A group of lanes takes up to
// eight rows in a line: heads of one token, whose angles are fetched once for them, or, of a tensor with one head,
// neighbouring tokens; so that what a row costs beyond its arithmetic is a step of a pointer.  All of a call's tensors go in one launch, each with its own range of blocks.  The backward keeps the columns of
// dw that a lane owns in registers over all rows that it visits and has the next rows on their way while it works;
// blocks write their sums to a plane each, which a second kernel adds in a fixed order, so that repeated calls agree to
// the bit.  Measured on 4 x 8192 tokens of 10 heads of 128, BF16: forward 35 us = 4.8 TB/s, backward 65 us =
// 3.9 TB/s and 5 us for the sums of dw (a plain copy moves 6.55), bound by the latency of a row and the issue of its
// instructions.  The append of 16 prompts of up to 2000 tokens, 4 key heads of 128: 38 us = 3.4 TB/s; one token of 64
// sequences: 5 us, which is a launch and three loads that wait for one another.
#include <algorithm>

#include "att3_abi_internal.h"
#include "serve_common.cuh"
#include "sm100_ptx.cuh"

namespace {

using serve::Four;

__device__ int g_serve_status = 0;

constexpr int THREADS = 256;
constexpr int LINE = 8;                            // rows of an item, the unit of work of D / 8 lanes
constexpr int FWD_ROWS = 4;                        // rows in flight
constexpr int MAX_TENSORS = 5;
constexpr int FWD_BLOCKS_PER_SM = 32, BWD_BLOCKS_PER_SM = 6;       // at most; a block then takes several items a group

struct Tensor {
    const void* x;
    void* y;
    const void* dy;
    void* dx;
    const void* w;
    float* dw;
    long long xb, yb, dyb, dxb;                    // strides of the batch, then of the position and the head, in elements
    int xn, xh, yn, yh, dyn, dyh, dxn, dxh;
    int w_type, rotate, heads, block0, blocks;
    serve::Divide by_lines;                        // items of a token, or (one head) of a sequence
    int lines, items;
};

struct Params {
    Tensor t[MAX_TENSORS];
    int n;
    const float* table;
    const void* positions;
    long long pos_b, pos_n;
    int pos_bytes, table_rows, rot, interleaved;
    int B, N;
    serve::Divide by_N;
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

// A lane's eight columns: four from `a` on, four from `b` on.  Of the rotated columns lane l has the pairs with the
// angles 4 l .. 4 l + 3.
struct Columns { int a, b; bool turns; };
__device__ __forceinline__ Columns columns_of(const Params& p, int lane_in_row) {
    const bool turns = lane_in_row * 8 < p.rot;
    if (turns && !p.interleaved) return Columns{lane_in_row * 4, (p.rot >> 1) + lane_in_row * 4, true};
    return Columns{lane_in_row * 8, lane_in_row * 8 + 4, turns};
}

template <typename T>
struct Row8 {
    Four<T> a, b;
    __device__ __forceinline__ void load(const T* p, const Columns& c) { a.load(p + c.a); b.load(p + c.b); }
    __device__ __forceinline__ void get(float (&f)[8]) const { a.get(f); b.get(f + 4); }
    static __device__ __forceinline__ void store(T* p, const Columns& c, const float (&f)[8]) {
        Four<T>::store(p + c.a, f);
        Four<T>::store(p + c.b, f + 4);
    }
};

__device__ __forceinline__ void load_scale(const Tensor& t, const Columns& c, float (&w)[8]) {
    if (t.w_type == 0) { Row8<__nv_bfloat16> v; v.load(static_cast<const __nv_bfloat16*>(t.w), c); v.get(w); }
    else if (t.w_type == 1) { Row8<__half> v; v.load(static_cast<const __half*>(t.w), c); v.get(w); }
    else { Row8<float> v; v.load(static_cast<const float*>(t.w), c); v.get(w); }
}

// Two FP32 at a time: f[k] * by[k] of eight, and sums of eight products.
__device__ __forceinline__ void scale8(float (&f)[8], const float (&by)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += 2) sm100::unpair_f32(sm100::mul_f32x2(sm100::pair_f32(f[k], f[k + 1]), sm100::pair_f32(by[k], by[k + 1])), f[k], f[k + 1]);
}
__device__ __forceinline__ void scale8(float (&f)[8], float by) {
#pragma unroll
    for (int k = 0; k < 8; k += 2) sm100::unpair_f32(sm100::mul_f32x2(sm100::pair_f32(f[k], f[k + 1]), sm100::pair_f32(by, by)), f[k], f[k + 1]);
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
    uint64_t s = sm100::mul_f32x2(sm100::pair_f32(a[0], a[1]), sm100::pair_f32(b[0], b[1]));
#pragma unroll
    for (int k = 2; k < 8; k += 2) s = sm100::fma_f32x2(sm100::pair_f32(a[k], a[k + 1]), sm100::pair_f32(b[k], b[k + 1]), s);
    float x, y;
    sm100::unpair_f32(s, x, y);
    return x + y;
}

// A lane's four angles (cosines 1, sines 0 where it turns nothing).
struct Angles { float4 c, s; };
__device__ __forceinline__ Angles load_angles(const Params& p, int pos, int lane_in_row, bool turns) {
    Angles t{make_float4(1.f, 1.f, 1.f, 1.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    if (turns) {
        const float* row = p.table + static_cast<long long>(pos) * p.rot + lane_in_row * 4;
        t.c = *reinterpret_cast<const float4*>(row);
        t.s = *reinterpret_cast<const float4*>(row + (p.rot >> 1));
    }
    return t;
}
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}
// Rot y (sign = 1) or Rot^T y (sign = -1), in place.
__device__ __forceinline__ void rotate(bool interleaved, float (&y)[8], const Angles& t, float sign) {
    const float c[4] = {t.c.x, t.c.y, t.c.z, t.c.w}, s[4] = {sign * t.s.x, sign * t.s.y, sign * t.s.z, sign * t.s.w};
    if (interleaved) {
#pragma unroll
        for (int k = 0; k < 4; ++k) turn(y[2 * k], y[2 * k + 1], c[k], s[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint64_t a = sm100::pair_f32(y[k], y[k + 1]), b = sm100::pair_f32(y[k + 4], y[k + 5]);
            const uint64_t cc = sm100::pair_f32(c[k], c[k + 1]), ss = sm100::pair_f32(s[k], s[k + 1]), minus = sm100::pair_f32(-s[k], -s[k + 1]);
            sm100::unpair_f32(sm100::fma_f32x2(b, minus, sm100::mul_f32x2(a, cc)), y[k], y[k + 1]);
            sm100::unpair_f32(sm100::fma_f32x2(a, ss, sm100::mul_f32x2(b, cc)), y[k + 4], y[k + 5]);
        }
    }
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

// The first row of an item and how many it has; the following ones are the next heads or, of a tensor with ONE head, the
// next positions.
struct Place { int b, n, head, rows; };
template <bool ONE>
__device__ __forceinline__ Place place_of(const Params& p, const Tensor& t, int item) {
    const int outer = t.by_lines(item), start = (item - outer * t.lines) * LINE;
    if (ONE) return Place{outer, start, 0, min(LINE, p.N - start)};
    const int b = p.by_N(outer);
    return Place{b, outer - b * p.N, start, min(LINE, t.heads - start)};
}

__device__ __forceinline__ int position_of(const Params& p, int b, int n) {
    long long pos = n;
    if (p.positions) {
        const long long at = b * p.pos_b + n * p.pos_n;
        pos = p.pos_bytes == 8 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
    }
    if (pos < 0 || pos >= p.table_rows) {
        serve::report(p.status, serve::ST_POSITION);
        pos = 0;
    }
    return static_cast<int>(pos);
}

// PAGED: the results of all tensors but the fifth (the queries) go to the cache rows of slot lengths[b] + n, and that
// slot is the position unless `positions` names the position of the first new token.
template <typename XT, int D, bool PAGED, bool ONE>
__device__ __forceinline__ void forward_rows(const Params& p, const Tensor& t, int ti) {
    constexpr int LANES = D / 8, GROUPS = THREADS / LANES;
    const int lr = threadIdx.x % LANES;
    const Columns cols = columns_of(p, lr);
    const bool turns = t.rotate && cols.turns, normed = t.w != nullptr, interleaved = p.interleaved != 0;
    const bool to_cache = PAGED && ti < 4;
    const float eps = p.eps;
    const long long step_x = ONE ? t.xn : t.xh, step_y = to_cache ? D : ONE ? t.yn : t.yh;
    __nv_bfloat16* const y0 = static_cast<__nv_bfloat16*>(t.y);
    float w[8];
    if (normed) load_scale(t, cols, w);
    const int items = t.items, stride = t.blocks * GROUPS;
    // every lane of a warp makes the same number of turns: the shuffles want all of them
    for (int base = (blockIdx.x - t.block0) * GROUPS; base < items; base += stride) {
        const int item = base + threadIdx.x / LANES;
        Place at{0, 0, 0, 0};
        if (item < items) at = place_of<ONE>(p, t, item);
        const XT* x = static_cast<const XT*>(t.x) + at.b * t.xb + static_cast<long long>(at.n) * t.xn + static_cast<long long>(at.head) * t.xh;
        // where the rows go, and the position of the first
        __nv_bfloat16* y = y0 + at.b * t.yb + static_cast<long long>(at.n) * t.yn + static_cast<long long>(at.head) * t.yh;
        int slot = 0, told = LINE;                         // the first row's slot in the cache; positions that a count covers
        long long first = 0;
        if (PAGED && at.rows > 0) {
            slot = p.lengths[at.b] + at.n;
            first = p.positions ? static_cast<long long>(static_cast<const int*>(p.positions)[at.b]) + at.n : slot;
            if (p.counts) {
                told = p.counts[at.b] - at.n;
                if (to_cache) at.rows = ONE ? max(0, min(at.rows, told)) : told > 0 ? at.rows : 0;       // what is not stored is not read
            }
        }
        auto position = [&](int u) {                       // of row u
            if (!PAGED) return position_of(p, at.b, at.n + (ONE ? u : 0));
            const long long q = first + (ONE ? u : 0);
            if (q >= 0 && q < p.table_rows) return static_cast<int>(q);
            if ((ONE ? u : 0) < told) serve::report(p.status, serve::ST_POSITION);          // a query behind the count may lie anywhere
            return 0;
        };
        auto cached = [&](int u) -> __nv_bfloat16* {       // the cache's row of token u, head `at.head`; none where it has no page
            const int row = p.pages.row(at.b, slot + u);
            if (row >= 0) return y0 + static_cast<long long>(row) * p.Hkv * D + at.head * D;
            serve::report(p.status, serve::ST_PAGE);
            return nullptr;
        };
        Angles angles;
        if (!ONE) {
            angles = load_angles(p, turns && at.rows > 0 ? position(0) : 0, lr, turns);
            if (to_cache) y = at.rows > 0 ? cached(0) : nullptr;
        }
        const int line = ONE ? LINE : min(LINE, t.heads);  // the same for the whole block
#pragma unroll 1
        for (int r = 0; r < line; r += FWD_ROWS) {
            Row8<XT> raw[FWD_ROWS];
#pragma unroll
            for (int u = 0; u < FWD_ROWS; ++u)
                if (r + u < at.rows) raw[u].load(x + (r + u) * step_x, cols);
#pragma unroll
            for (int u = 0; u < FWD_ROWS; ++u) {
                const bool here = r + u < at.rows;
                if (ONE && turns) angles = load_angles(p, here ? position(r + u) : 0, lr, true);
                float f[8];
                if (here) raw[u].get(f);
                else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] = 0.f;
                }
                if (normed) {
                    const float q = rsqrtf(row_sum<LANES>(dot8(f, f)) * (1.f / D) + eps);
                    scale8(f, q);
                    scale8(f, w);
                }
                if (turns) rotate(interleaved, f, angles, 1.f);
                if (!here) continue;
                __nv_bfloat16* to = ONE && to_cache ? cached(r + u) : to_cache && !y ? nullptr : y + (r + u) * step_y;
                if (!to) continue;
                Row8<__nv_bfloat16>::store(to, cols, f);
                if (PAGED && ti == 0 && p.mass && lr == 0) p.mass[(to - y0) / D] = 0.f;
            }
        }
    }
}

template <typename XT, int D, bool PAGED>
__global__ void __launch_bounds__(THREADS, sizeof(XT) == 2 ? 4 : 3) norm_rotate_kernel(const __grid_constant__ Params p) {
    serve::wait_for_previous_kernel();
    const int ti = find_tensor(p);
    const Tensor& t = p.t[ti];
    if (t.heads == 1) forward_rows<XT, D, PAGED, true>(p, t, ti);
    else forward_rows<XT, D, PAGED, false>(p, t, ti);
}

// Adds the rows' share of dw to `dw`, a lane its eight columns.
template <typename XT, int D, bool ONE>
__device__ __forceinline__ void backward_rows(const Params& p, const Tensor& t, const Columns& cols, int lr, float (&dw)[8]) {
    // rows in flight: registers go further with four of 16 bits and two blocks an SM than with two and three (65 us against
    // 77 for 32768 tokens of 10 heads of 128); FP32 rows the other way round (37 against 25 for 8188 tokens of 24 of 64)
    constexpr int BWD_ROWS = sizeof(XT) == 2 ? 4 : 2;
    constexpr int LANES = D / 8, GROUPS = THREADS / LANES;
    const bool turns = t.rotate && cols.turns, normed = t.w != nullptr, interleaved = p.interleaved != 0;
    const float eps = p.eps;
    const long long step_x = ONE ? t.xn : t.xh, step_g = ONE ? t.dyn : t.dyh, step_d = ONE ? t.dxn : t.dxh;
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = 1.f;
    if (normed) load_scale(t, cols, w);
    const int items = t.items, stride = t.blocks * GROUPS, line = ONE ? LINE : min(LINE, t.heads);
    // every lane of a warp makes the same number of turns: the shuffles want all of them
    for (int base = (blockIdx.x - t.block0) * GROUPS; base < items; base += stride) {
        const int item = base + threadIdx.x / LANES;
        Place at{0, 0, 0, 0};
        if (item < items) at = place_of<ONE>(p, t, item);
        const XT* x = static_cast<const XT*>(t.x) + at.b * t.xb + static_cast<long long>(at.n) * t.xn + static_cast<long long>(at.head) * t.xh;
        const __nv_bfloat16* dy = static_cast<const __nv_bfloat16*>(t.dy) + at.b * t.dyb + static_cast<long long>(at.n) * t.dyn +
                                  static_cast<long long>(at.head) * t.dyh;
        XT* dx = static_cast<XT*>(t.dx) + at.b * t.dxb + static_cast<long long>(at.n) * t.dxn + static_cast<long long>(at.head) * t.dxh;
        Row8<XT> next_x[BWD_ROWS];
        Row8<__nv_bfloat16> next_g[BWD_ROWS];
        auto fetch = [&](int r) {
#pragma unroll
            for (int u = 0; u < BWD_ROWS; ++u)
                if (r + u < at.rows) {
                    next_g[u].load(dy + (r + u) * step_g, cols);
                    if (normed) next_x[u].load(x + (r + u) * step_x, cols);
                }
        };
        fetch(0);
        Angles angles;
        if (!ONE) angles = load_angles(p, turns && at.rows > 0 ? position_of(p, at.b, at.n) : 0, lr, turns);
#pragma unroll 1
        for (int r = 0; r < line; r += BWD_ROWS) {
            Row8<XT> now_x[BWD_ROWS];
            Row8<__nv_bfloat16> now_g[BWD_ROWS];
#pragma unroll
            for (int u = 0; u < BWD_ROWS; ++u) { now_x[u] = next_x[u]; now_g[u] = next_g[u]; }
            fetch(r + BWD_ROWS);
#pragma unroll
            for (int u = 0; u < BWD_ROWS; ++u) {
                const bool here = r + u < at.rows;
                if (ONE && turns) angles = load_angles(p, here ? position_of(p, at.b, at.n + r + u) : 0, lr, true);
                float g[8], v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) g[k] = v[k] = 0.f;
                if (here) {
                    now_g[u].get(g);
                    if (normed) now_x[u].get(v);
                }
                if (turns) rotate(interleaved, g, angles, -1.f);
                if (normed) {
                    float wg[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) wg[k] = g[k];
                    scale8(wg, w);
                    const float ss = row_sum<LANES>(dot8(v, v)), m = row_sum<LANES>(dot8(v, wg));
                    const float q = here ? rsqrtf(ss * (1.f / D) + eps) : 0.f;          // with eps = 0 infinite: no row, no share of dw
                    const uint64_t qq = sm100::pair_f32(q, q);
                    const float f1 = -q * q * (m * q) * (1.f / D);
                    const uint64_t ff = sm100::pair_f32(f1, f1);
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        const uint64_t vv = sm100::pair_f32(v[k], v[k + 1]);
                        sm100::unpair_f32(sm100::fma_f32x2(sm100::pair_f32(g[k], g[k + 1]), sm100::mul_f32x2(vv, qq), sm100::pair_f32(dw[k], dw[k + 1])),
                                          dw[k], dw[k + 1]);
                        sm100::unpair_f32(sm100::fma_f32x2(vv, ff, sm100::mul_f32x2(qq, sm100::pair_f32(wg[k], wg[k + 1]))), g[k], g[k + 1]);
                    }
                }
                if (here) Row8<XT>::store(dx + (r + u) * step_d, cols, g);
            }
        }
    }
}

template <typename XT, int D>
__global__ void __launch_bounds__(THREADS, 2) norm_rotate_backward_kernel(const __grid_constant__ Params p) {
    constexpr int LANES = D / 8, GROUPS = THREADS / LANES;
    __shared__ float sums[GROUPS][D];
    serve::wait_for_previous_kernel();
    const Tensor& t = p.t[find_tensor(p)];
    const int lr = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const Columns cols = columns_of(p, lr);
    float dw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t.heads == 1) backward_rows<XT, D, true>(p, t, cols, lr, dw);
    else backward_rows<XT, D, false>(p, t, cols, lr, dw);
    if (!t.w) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        sums[group][cols.a + k] = dw[k];
        sums[group][cols.b + k] = dw[k + 4];
    }
    __syncthreads();
    if (threadIdx.x < D) {
        float a = 0.f;
        for (int q = 0; q < GROUPS; ++q) a += sums[q][threadIdx.x];
        p.partial[static_cast<long long>(blockIdx.x) * D + threadIdx.x] = a;
    }
}

// dw of 16 columns of one tensor: the planes of its blocks, added in a fixed order (64 shares, then those).
constexpr int GRAD_COLS = 16, GRAD_PARTS = 64;
__global__ void __launch_bounds__(GRAD_COLS * GRAD_PARTS) scale_grad_kernel(const __grid_constant__ Params p, int D) {
    __shared__ float sums[GRAD_PARTS][GRAD_COLS];
    const Tensor& t = p.t[blockIdx.x];
    serve::wait_for_previous_kernel();
    if (!t.w) return;
    const int c = threadIdx.x % GRAD_COLS, part = threadIdx.x / GRAD_COLS, col = blockIdx.y * GRAD_COLS + c;
    float a = 0.f;
#pragma unroll 8
    for (int q = part; q < t.blocks; q += GRAD_PARTS) a += p.partial[static_cast<long long>(t.block0 + q) * D + col];
    sums[part][c] = a;
    __syncthreads();
    if (part == 0) {
#pragma unroll 16
        for (int q = 1; q < GRAD_PARTS; ++q) a += sums[q][c];
        t.dw[col] = a;
    }
}

size_t element(int type) { return type == 2 ? 4 : 2; }

bool aligned(const void* ptr, const int64_t* strides, int type) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return false;
    for (int k = 0; strides && k < 3; ++k)
        if ((k > 0 && (strides[k] > 0x7FFFFFFFll || strides[k] < 0)) || strides[k] * static_cast<int64_t>(element(type)) % 16 != 0) return false;
    return true;
}

// Checks and fills what forward, backward and append have in common.  Blocks of a tensor: one group per item, but no
// more than its share of `budget` blocks in proportion to its rows.
int fill(Params& p, const char* who, const att3_head_rows* t, int n, int x_type, const float* table, int table_rows,
         int rot, int interleaved, int B, int N, int D, float eps, int budget) {
    if (!t || n < 1 || n > MAX_TENSORS) return att3::set_error(ATT3_ERR_INVALID, "%s: 1 to %d tensors, got %d", who, MAX_TENSORS, n);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return att3::set_error(ATT3_ERR_INVALID, "%s: head dim must be 16, 32, 64 or 128, got %d", who, D);
    if (B < 0 || N < 0) return att3::set_error(ATT3_ERR_INVALID, "%s: negative batch or length", who);
    if (x_type < 0 || x_type > 2) return att3::set_error(ATT3_ERR_INVALID, "%s: unknown element type %d", who, x_type);
    if (!(eps >= 0.f)) return att3::set_error(ATT3_ERR_INVALID, "%s: eps must not be negative", who);
    if (rot < 0 || rot > D || rot % 8 != 0)
        return att3::set_error(ATT3_ERR_INVALID, "%s: rotated columns must be a multiple of 8 up to the head dim %d, got %d", who, D, rot);
    if (rot && (!table || table_rows < 1 || reinterpret_cast<uintptr_t>(table) % 16 != 0))
        return att3::set_error(ATT3_ERR_INVALID, "%s: the rotation needs a 16-byte aligned table with at least one row", who);
    p.n = n;
    p.table = table;
    p.table_rows = table_rows;
    p.rot = rot;
    p.interleaved = interleaved != 0;
    p.B = B;
    p.N = N;
    p.by_N = serve::make_divide(std::max(1, N));
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
        o.xb = t[k].x_stride[0]; o.yb = t[k].y_stride[0]; o.dyb = t[k].dy_stride[0]; o.dxb = t[k].dx_stride[0];
        o.xn = static_cast<int>(t[k].x_stride[1]); o.xh = static_cast<int>(t[k].x_stride[2]);
        o.yn = static_cast<int>(t[k].y_stride[1]); o.yh = static_cast<int>(t[k].y_stride[2]);
        o.dyn = static_cast<int>(t[k].dy_stride[1]); o.dyh = static_cast<int>(t[k].dy_stride[2]);
        o.dxn = static_cast<int>(t[k].dx_stride[1]); o.dxh = static_cast<int>(t[k].dx_stride[2]);
        if (o.w && (o.w_type < 0 || o.w_type > 2)) return att3::set_error(ATT3_ERR_INVALID, "%s: unknown element type of scale %d", who, k);
        if (o.w && reinterpret_cast<uintptr_t>(o.w) % 16 != 0) return att3::set_error(ATT3_ERR_INVALID, "%s: scale %d must be 16-byte aligned", who, k);
        o.heads = static_cast<int>(t[k].heads);
        // one head: lines of positions; more heads: lines of a token's heads
        o.lines = static_cast<int>((static_cast<long long>(o.heads == 1 ? N : o.heads) + LINE - 1) / LINE);
        o.by_lines = serve::make_divide(std::max(1, o.lines));
        const long long outer = o.heads == 1 ? B : static_cast<long long>(B) * N, items = outer * o.lines;
        if (static_cast<long long>(B) * N * o.heads > 0x3FFFFFFFll) return att3::set_error(ATT3_ERR_INVALID, "%s: more than 2^30 rows in a tensor", who);
        o.items = static_cast<int>(items);
        long long nb = (items + groups - 1) / groups;
        nb = std::min(nb, std::max<long long>(1, budget * static_cast<long long>(o.heads) / rows));
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
    att3::count_launch(4);
    const att3::TimedLaunch timed(att3::K_SERVE, st);
    cudaError_t e = cudaSuccess;
#define ATT3_NR(T, DD) e = serve::launch_early(norm_rotate_kernel<T, DD, PAGED>, dim3(blocks), dim3(THREADS), 0, st, p)
#define ATT3_NR_D(T) do { if (D == 16) ATT3_NR(T, 16); else if (D == 32) ATT3_NR(T, 32); else if (D == 64) ATT3_NR(T, 64); else ATT3_NR(T, 128); } while (0)
    if (x_type == 0) ATT3_NR_D(__nv_bfloat16);
    else if (x_type == 1) ATT3_NR_D(__half);
    else ATT3_NR_D(float);
#undef ATT3_NR_D
#undef ATT3_NR

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
    if (int rc = fill(p, who, tensors, n, x_type, table, table_rows, rot, interleaved, B, N, D, eps, att3::sm_count() * FWD_BLOCKS_PER_SM)) return rc;
    if (positions && pos_bytes != 4 && pos_bytes != 8) return att3::set_error(ATT3_ERR_INVALID, "%s: positions are 4 or 8 bytes wide", who);
    if (B == 0 || N == 0) return ATT3_OK;
    for (int k = 0; k < n; ++k) {
        if (!tensors[k].x || !tensors[k].y) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor %d", who, k);
        if (!aligned(tensors[k].x, tensors[k].x_stride, x_type) || !aligned(tensors[k].y, tensors[k].y_stride, 0))
            return att3::set_error(ATT3_ERR_INVALID, "%s: rows of tensor %d must be 16-byte aligned, with strides below 2^31", who, k);
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
    att3::count_launch(4, (blocks ? 1 : 0) + (scaled ? 1 : 0));
    const att3::TimedLaunch timed(att3::K_SERVE, st);
    cudaError_t e = cudaSuccess;
    if (blocks) {
#define ATT3_NR(T, DD) e = serve::launch_early(norm_rotate_backward_kernel<T, DD>, dim3(blocks), dim3(THREADS), 0, st, p)
#define ATT3_NR_D(T) do { if (D == 16) ATT3_NR(T, 16); else if (D == 32) ATT3_NR(T, 32); else if (D == 64) ATT3_NR(T, 64); else ATT3_NR(T, 128); } while (0)
        if (x_type == 0) ATT3_NR_D(__nv_bfloat16);
        else if (x_type == 1) ATT3_NR_D(__half);
        else ATT3_NR_D(float);
#undef ATT3_NR_D
#undef ATT3_NR
    }
    // with no rows at all this writes the gradient's zeros
    if (e == cudaSuccess && scaled)
        e = serve::launch_early(scale_grad_kernel, dim3(n, D / GRAD_COLS), dim3(GRAD_COLS * GRAD_PARTS), 0, st, p, D);
    return e == cudaSuccess ? ATT3_OK : att3::set_cuda_error(e, who);
}

extern "C" int att3_gather_cache_append(const att3_head_rows* tensors, int n, int x_type, const float* table, int table_rows,
                                        int rot, int interleaved, const int* positions, const att3_gather_pages* pages,
                                        const int* lengths, const int* counts, float* mass, int B, int T, int D, float eps,
                                        void* stream) {
    const char* who = "att3_gather_cache_append";
    Params p = {};
    if (n != 4 && n != 5) return att3::set_error(ATT3_ERR_INVALID, "%s: R, S, Vr, Vs and optionally Q, got %d tensors", who, n);
    if (int rc = fill(p, who, tensors, n, x_type, table, table_rows, rot, interleaved, B, T, D, eps, att3::sm_count() * FWD_BLOCKS_PER_SM)) return rc;
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
