// The single gather of one new token over a paged gather cache, sm_100a.
//
// For one query head, with E visible slots e (the first `sinks`, the last `window`, or all),
//
//     x_jk = sum_d q_d r_jd s_kd / sqrt(D),   p = softmax over all pairs (j, k),   y_d = sum_jk p_jk vr_jd vs_kd.
//
// Read as a tile product the pairs are a matrix: rows (q o R_j), columns S_k.  X = (q o R) S^T, P = exp(X - m),
// U = P Vs are two tensor-core products of 128 x 128 tiles, and y collapses the rows, y = sum_j Vr_j o U_j.  This is
// 4 D E^2 operations a head on 8 D E bytes a key head: bound by the tensor cores for long caches (64 and more keys a
// head already do 256 operations a byte with 8 heads a key head), by latency for a few hundred pairs.
//
// Scores.  q o R is not rounded: a BF16 x BF16 product has at most 16 significant bits, so its BF16 value and the
// BF16 residual carry it exactly, and the score is the sum of two products in FP32.  That makes 1.5 times the matrix
// work of the rounded form; what it buys is that the softmax, the token masses and the comparison with the prompt's
// pass do not depend on the size of the scores.  P is rounded to BF16 for the second product, as in the prompt's
// kernels; its sums stay FP32.
//
// Strips.  A strip is 32 keys of one query head, and one warp's; a CTA works on tiles of eight strips, two halves of
// 128 rows with a tensor-memory accumulator each.  The query heads of a key head are taken in blocks of 8, 4, 2 and 1,
// and a block's strips in the order of their keys, all its heads side by side: a tile of eight heads reads 32 rows of R
// and Vr once for all of them, a short cache fills its tiles with several heads, and a warp stays with one head through
// a block.  A strip's maximum is the warp's: the softmax of a head is joint over all its pairs, so rows far below the
// strip's maximum may underflow as they would in the end.
//
// Splits.  The unit of work is (sequence, key head, tile, 128 keys).  All units lie on one line, each CTA takes an
// equal stretch of it (one CTA an SM), and a stretch may begin and end inside a tile's key loop: any mix of lengths
// keeps every SM busy, and one long sequence is split over its keys.  The lengths are read on the device, so a
// captured graph follows them.  A warp carries (y, m, l) along its strips of one head and writes them out when its
// stretch leaves the head; decode_join_kernel brings the partials of a head together in a fixed order.
//
// Roles.  Warps 0-3 and 4-7: one half each -- build the two operand tiles of q o R, exponentials, collapse.  Warp 8
// issues the products, warps 9-11 bring S and Vs rows through the page table into a ring of stages by TMA: whole boxes
// of a page where every slot is visible (no window, a full key step), else row gathers, four rows an instruction, for
// which neither the page size nor where a window begins matters.  Issuing is what costs: a tile of 128 rows of 128
// takes 4200 cycles as row gathers from one warp (62 an instruction), 1700 from three, 930 as boxes of 16 rows and 720
// as boxes of 64; 16-byte asynchronous copies from three warps took 2060.  While one half exponentiates, the other
// half's products run.
//
// Tensor memory: per half 128 columns of scores, over which P is written, then 128 of U.  Where no sequence shows more
// than 192 slots (a window of 128 with a few sinks), a tile's keys are one step: its scores run on into the columns of U,
// which nothing is in before the step's second product, and a stage of the ring holds 192 rows.  Without that, 132 visible
// slots take two steps, the second for four columns.
//
// Masses (a token's share of the attention) need column sums of P too: a lane has a row, so 32 columns cost an exchange of
// 31 shuffles, and the four warps of a half add theirs up through shared memory.  A CTA keeps the sums of a head over all
// the tiles that it goes through, relative to the largest maximum so far; decode_mass_kernel puts them together once the
// head's sum is known.
//
// Measured, calls among others, in short runs and (in brackets) in long ones, where the power cap lowers the clock: 2
// sequences of 8191 keys, 8 heads of 128: 562 us (650), 980 TFLOP/s of the formula's operations and 1470 of the products
// issued, bound by the tensor pipe and the shared memory that feeds it; 16 sequences of up to 2000 keys, 8 heads of 64: 120
// us (134-160), the exponentials; 4 of up to 2500 keys with masses: 111 us (119-124), 15 us of them the join and the masses;
// 128 sequences with 132 visible slots, 8 heads of 128: 44.7 us, and one sequence with 128: 12.2 us, the chain from row
// addresses to the collapse.
#pragma once

#include "att3_abi_internal.h"
#include "serve_common.cuh"
#include "sg_ring_common.cuh"

namespace serve {

using namespace sm100;
using sgring::warp_arrive;

constexpr int DEC_THREADS = 384;
constexpr int DEC_STRIP = 32;              // rows of a strip
constexpr int DEC_TILE_STRIPS = 8;
constexpr int DEC_KEYS = 128;              // keys of a unit of work
constexpr int DEC_WIDE = 192;              // of the only unit of a tile, where no sequence shows more (DecodeParams::wide)
constexpr int DEC_COPY_WARPS = 3;

struct DecodeParams {
    const __nv_bfloat16* Q;                // [B,Hq,D]
    const __nv_bfloat16* R;                // pools
    const __nv_bfloat16* Vr;
    __nv_bfloat16* Y;                      // [B,Hq,D]
    float* mass;                           // [pages, page_size, Hkv] or null
    const int* lengths;
    Pages pages;
    int B, Hq, Hkv, G, window, sinks;
    float c2;                              // log2(e) / sqrt(D)
    // workspace
    float* part;                           // [head + CTA][8 warps] records of D + 4 floats: y, m, l
    float* rows;                           // mass: [tile + CTA][8 warps][32] row sums
    float* row_ref;                        // mass: [tile + CTA][8 warps] the maximum they are relative to
    float* cols;                           // mass: column sums, [head + CTA][2 halves][col_steps][128], or with `brief` [unit][8 strips][128]
    float* col_ref;                        // mass: the maximum that each 128 of them are relative to
    float* lse;                            // mass: [B,Hq] log2 of the softmax sum
    int* unit_base;                        // [B + 1]; the host admits no more than 2^31 - 1 units
    int* tile_base;                        // [B + 1]
    int* status;
    // pools as [pages * page_size, Hkv * D], 64 columns of one row, or of `box` rows of a page (0: not used)
    CUtensorMap tmS, tmVs, tmS_box, tmVs_box;
    int box;
    int col_steps;                         // key steps of the longest sequence
    int brief;                             // with masses, 1: no sequence shows more than 128 slots
    int wide;                              // 1: no sequence shows more than 192 slots, and a tile has one step of up to 192 keys
};

// Tiles of a block of `heads` (1, 2, 4 or 8) heads with `groups` strips each.
__device__ __forceinline__ int block_tiles(int heads, int groups) { return (heads * groups + DEC_TILE_STRIPS - 1) / DEC_TILE_STRIPS; }

// What one sequence's work looks like.
struct Shape {
    int n, seen, skip;                     // length, visible slots, slots between the sinks and the window
    int groups, tiles, steps;              // strips of a head; tiles of a key head; key steps
    __device__ __forceinline__ int units(int Hkv) const { return Hkv * tiles * steps; }
};

template <bool MASS>
__device__ __forceinline__ Shape shape_of(const DecodeParams& p, int b, bool tell = false) {
    Shape s;
    s.n = p.pages.length(p.lengths, b, p.status, tell);
    s.seen = p.window > 0 ? min(s.n, p.window + p.sinks) : s.n;
    s.skip = s.n - s.seen;
    s.groups = (s.seen + DEC_STRIP - 1) / DEC_STRIP;
    if (MASS && !p.brief) s.tiles = p.G * block_tiles(1, s.groups);
    else s.tiles = p.G / 8 * s.groups + (p.G & 4 ? block_tiles(4, s.groups) : 0) + (p.G & 2 ? block_tiles(2, s.groups) : 0) +
                   (p.G & 1 ? block_tiles(1, s.groups) : 0);
    s.steps = p.wide ? min(s.seen, 1) : (s.seen + DEC_KEYS - 1) / DEC_KEYS;
    return s;
}

// A block of query heads: `heads` of them from g0 on (inside the key head), its tiles from tile0 on.  With masses every
// block is one head, so that a half's column sums are one head's and can be added up, over the strips of a tile and over the
// tiles that a CTA goes through (so they take memory by the slot, not by the pair); but where a tile has one key step
// at most (`brief`) they are kept strip by strip and heads share tiles as without masses (8 heads a key head, 128 key
// heads: at window 16, one tile in place of eight, 66 -> 27 us, at window 128 72 -> 55).
struct Block { int g0, log_heads, tile0; };

template <bool MASS>
__device__ __forceinline__ Block block_of_tile(const DecodeParams& p, const Shape& s, int tile) {
    if (MASS && !p.brief) {
        const int per = block_tiles(1, s.groups), g = tile / per;
        return Block{g, 0, g * per};
    }
    const int eights = p.G / 8, whole = eights * s.groups;
    if (tile < whole) {
        const int k = eights == 1 ? 0 : tile / s.groups;
        return Block{8 * k, 3, k * s.groups};
    }
    Block k{8 * eights, 2, whole};
    if (p.G & 4) {
        const int n = block_tiles(4, s.groups);
        if (tile < k.tile0 + n) return k;
        k.g0 += 4;
        k.tile0 += n;
    }
    k.log_heads = 1;
    if (p.G & 2) {
        const int n = block_tiles(2, s.groups);
        if (tile < k.tile0 + n) return k;
        k.g0 += 2;
        k.tile0 += n;
    }
    k.log_heads = 0;
    return k;
}

template <bool MASS>
__device__ __forceinline__ Block block_of_head(const DecodeParams& p, const Shape& s, int g) {
    if (MASS && !p.brief) return Block{g, 0, g * block_tiles(1, s.groups)};
    const int eights = p.G / 8;
    if (g < 8 * eights) return Block{g & ~7, 3, g / 8 * s.groups};
    Block k{8 * eights, 2, eights * s.groups};
    if (p.G & 4) {
        if (g < k.g0 + 4) return k;
        k.g0 += 4;
        k.tile0 += block_tiles(4, s.groups);
    }
    k.log_heads = 1;
    if (p.G & 2) {
        if (g < k.g0 + 2) return k;
        k.g0 += 2;
        k.tile0 += block_tiles(2, s.groups);
    }
    k.log_heads = 0;
    return k;
}

__device__ __forceinline__ int slot_of(const DecodeParams& p, const Shape& s, int e) {
    return p.window > 0 && e >= p.sinks ? e + s.skip : e;
}

// The stretch of CTA c of n begins at unit stretch(total, c, n): the first total % n of them have one unit more.
__device__ __forceinline__ int stretch(int total, int c, int n) {
    const int per = total / n;
    return c * per + min(c, total - per * n);
}
// The CTA whose stretch holds `unit`.
__device__ __forceinline__ int cta_of(int unit, int total, int n) {
    const int per = total / n, more = total - per * n, head = more * (per + 1);
    return unit < head ? unit / (per + 1) : more + (unit - head) / per;
}

// A CTA's way along its stretch, one tile's key range at a time; every role walks it by itself.
template <bool MASS>
struct Walk {
    Shape s;
    int b, head, tile, k0, k1;             // sequence, key head, tile, key steps [k0, k1)
    int left, unit, slot;                  // units still to do, of the first step, row sums' slot
    Block block;                           // of the tile, and the tile behind it
    int block_end;
    int first_tile, first_k;               // where the CTA came into the block
    __device__ __forceinline__ void enter(const DecodeParams& p) {
        block = block_of_tile<MASS>(p, s, tile);
        block_end = block.tile0 + block_tiles(1 << block.log_heads, s.groups);
        first_tile = tile;
        first_k = 0;
    }
    __device__ __forceinline__ void start(const DecodeParams& p, int b0, int off, int count, int tile_base, int unit0) {
        b = b0;
        s = shape_of<MASS>(p, b);
        const int per = s.tiles * s.steps;
        head = off / per;
        const int r = off - head * per;
        tile = r / s.steps;
        k0 = r - tile * s.steps;
        left = count;
        unit = unit0;
        slot = tile_base + head * s.tiles + tile + blockIdx.x;
        k1 = min(s.steps, k0 + left);
        enter(p);
        first_k = k0;
    }
    // whether the CTA has been at key step k of this block before
    __device__ __forceinline__ bool again(int k) const { return tile > first_tile + (k < first_k ? 1 : 0); }
    // false when the stretch is done
    __device__ __forceinline__ bool next(const DecodeParams& p) {
        left -= k1 - k0;
        unit += k1 - k0;
        if (left <= 0) return false;
        k0 = 0;
        ++slot;
        if (++tile == block_end) {
            if (tile == s.tiles) {
                tile = 0;
                if (++head == p.Hkv) {
                    head = 0;
                    do { ++b; if (b >= p.B) return false; s = shape_of<MASS>(p, b); } while (s.seen == 0);
                }
            }
            enter(p);
        }
        k1 = min(s.steps, left);
        return true;
    }
    // whether a half of the tile holds any key
    __device__ __forceinline__ bool live(int half) const {
        return (((tile - block.tile0) * DEC_TILE_STRIPS + half * 4) >> block.log_heads) < s.groups;
    }
    // columns of key step k in chunks of 32 (the last step's tiles and products are cut to them)
    template <bool WIDE>
    __device__ __forceinline__ int chunks(int k) const {
        return min((WIDE ? DEC_WIDE : DEC_KEYS) / 32, (s.seen - k * DEC_KEYS + 31) / 32);
    }
};

template <int D>
struct DecSmem {
    static constexpr int TILE = 128 * D * 2;                   // one [128][D] BF16 operand tile
    static constexpr int STAGES = D == 128 ? 3 : 8;
    static constexpr int OFF_A = 0;                            // [half][value, residual]
    static constexpr int OFF_KV = 4 * TILE;
    static constexpr int OFF_COL = OFF_KV + STAGES * TILE;     // mass: [half][2][128] column sums being added up
    static constexpr int OFF_SCAN = OFF_COL + 2048;            // per warp units and tiles, start of the stretch
    static constexpr int OFF_BARS = OFF_SCAN + 256;
    static constexpr int BYTES = OFF_BARS + 256;
    static_assert(BYTES <= 232448, "227 KB of shared memory");
};

enum DecBar { DB_A_FULL0 = 0, DB_A_FULL1, DB_S_FULL0, DB_S_FULL1, DB_P_FULL0, DB_P_FULL1, DB_O_DONE0, DB_O_DONE1, DB_DRAIN,
              DB_COL0, DB_COL1,
              DB_KV_FULL0, DB_KV_EMPTY0 = DB_KV_FULL0 + 8, DB_COUNT = DB_KV_EMPTY0 + 8 };

// Four rows (y) of 64 columns from x on, to four consecutive 128-byte lines.
__device__ __forceinline__ void tma_gather4(void* dst, const void* map, int x, const int (&y)[4], uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(smem_u32(bar))
        : "memory");
}

// Residual of a packed BF16 product hi = bf16x2(a b): a b - hi has at most 8 significant bits, so the fused
// multiply-add, which rounds once, gives it exactly.  Where the product itself is out of range the residual is NaN; the
// minimum, which prefers a number, makes it the largest that a residual can be, which changes nothing beside the infinite
// value (a NaN factor is in hi too).
__device__ __forceinline__ uint32_t residual_bf16x2(uint32_t a, uint32_t b, uint32_t hi) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b),
                                     __hneg2(*reinterpret_cast<const __nv_bfloat162*>(&hi)));
    const __nv_bfloat162 n = __hmin2(r, __float2bfloat162_rn(0x1p120f));
    return *reinterpret_cast<const uint32_t*>(&n);
}

// 16 bytes from global to shared memory, asynchronously; a thread's copies complete in groups.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A bounded wait whose outcome is the whole warp's: no lane goes on into a warp-wide instruction that another has left.
__device__ __forceinline__ bool pipe_wait(uint64_t* bar, uint32_t parity, volatile int* fail, int code) {
    return __all_sync(0xFFFFFFFFu, sgring::pipe_wait(bar, parity, fail, code));
}

// 16 lanes by 32 columns of tensor memory: lane L receives, for k = 0 .. 3, columns 8 k + 2 (L % 4), + 1 of row L / 4 in
// registers 4 k, 4 k + 1 and of row L / 4 + 8 in 4 k + 2, 4 k + 3.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

template <int D, bool MASS, bool WIDE>
__global__ void __launch_bounds__(DEC_THREADS, 1) decode_kernel(const __grid_constant__ DecodeParams p) {
    using L = DecSmem<D>;
    constexpr int REC = D + 4, COLS = D / 32;
    constexpr float GROW = 8.f;            // a strip's reference maximum is renewed when a score exceeds it by 2^8
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0) {   // the operand tiles' swizzle wants it; there is no room to align by hand
        wait_for_previous_kernel();
        if (threadIdx.x == 0) report(p.status, 10);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BARS);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_BARS + DB_COUNT * 8);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* sh_ref = reinterpret_cast<float*>(tmem_slot + 2);                   // [8]
    int (*sh_sum)[2] = reinterpret_cast<int (*)[2]>(smem + L::OFF_SCAN);
    int* sh_start = reinterpret_cast<int*>(smem + L::OFF_SCAN) + 2 * (DEC_THREADS / 32);
    static_assert((2 * (DEC_THREADS / 32) + 5) * 4 <= 256 && DB_COUNT * 8 + 8 + 32 <= 256, "shared bookkeeping");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- this CTA's stretch: units and tiles before every sequence, a run of sequences a thread
    int total;
    {
        if (tid == 0) {
            mbar_init(&bars[DB_A_FULL0], 4); mbar_init(&bars[DB_A_FULL1], 4);
            mbar_init(&bars[DB_S_FULL0], 1); mbar_init(&bars[DB_S_FULL1], 1);
            mbar_init(&bars[DB_P_FULL0], 4); mbar_init(&bars[DB_P_FULL1], 4);
            mbar_init(&bars[DB_O_DONE0], 1); mbar_init(&bars[DB_O_DONE1], 1);
            mbar_init(&bars[DB_DRAIN], 1);
            mbar_init(&bars[DB_COL0], 4); mbar_init(&bars[DB_COL1], 4);
            for (int x = 0; x < 8; ++x) { mbar_init(&bars[DB_KV_FULL0 + x], DEC_COPY_WARPS); mbar_init(&bars[DB_KV_EMPTY0 + x], 1); }
            fence_mbar_init();
            *fail = 0;
        }
        if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
        wait_for_previous_kernel();
        const int per = (p.B + DEC_THREADS - 1) / DEC_THREADS;
        const int lo = min(tid * per, p.B), hi = min(lo + per, p.B);
        int units = 0, tiles = 0;
        for (int b = lo; b < hi; ++b) {
            const Shape s = shape_of<MASS>(p, b, blockIdx.x == 0);
            units += s.units(p.Hkv);
            tiles += p.Hkv * s.tiles;
        }
        int iu = units, it = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int yu = __shfl_up_sync(0xFFFFFFFFu, iu, o), yt = __shfl_up_sync(0xFFFFFFFFu, it, o);
            if (lane >= o) { iu += yu; it += yt; }
        }
        if (lane == 31) { sh_sum[warp][0] = iu; sh_sum[warp][1] = it; }
        __syncthreads();
        int bu = 0, bt = 0, tt = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < DEC_THREADS / 32; ++w) {
            if (w < warp) { bu += sh_sum[w][0]; bt += sh_sum[w][1]; }
            total += sh_sum[w][0];
            tt += sh_sum[w][1];
        }
        bu += iu - units;
        bt += it - tiles;
        const int begin = stretch(total, blockIdx.x, gridDim.x), end = stretch(total, blockIdx.x + 1, gridDim.x);
        if (blockIdx.x == 0 && tid == 0) { p.unit_base[p.B] = total; p.tile_base[p.B] = tt; }
        if (blockIdx.x == 0 || (begin < end && begin >= bu && begin < bu + units)) {
            for (int b = lo; b < hi; ++b) {
                const Shape s = shape_of<MASS>(p, b);
                const int u = s.units(p.Hkv);
                if (blockIdx.x == 0) { p.unit_base[b] = bu; p.tile_base[b] = bt; }
                if (begin < end && begin >= bu && begin < bu + u) {
                    sh_start[0] = begin - bu;
                    sh_start[1] = end - begin;
                    sh_start[2] = bt;
                    sh_start[3] = begin;
                    sh_start[4] = b;
                }
                bu += u;
                bt += p.Hkv * s.tiles;
            }
        }
        if (tid == 0 && begin >= end) sh_start[4] = -1;
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }
    const uint32_t tmem = *tmem_slot;
    const bool busy = sh_start[4] >= 0;
    Walk<MASS> w;
    if (busy) w.start(p, sh_start[4], sh_start[0], sh_start[1], sh_start[2], sh_start[3]);

    if (warp < 8) {
        // ================================================================== builders, exponentials, collapse
        sgring::reg_inc<208>();
        const int half = warp >> 2, wq = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
        const uint32_t tS = tmem + lanes + half * 256, tO = tS + 128;
        uint8_t* tile_hi = smem + L::OFF_A + half * 2 * L::TILE;
        constexpr int CH = D / 8, RPP = 32 / CH, PASSES = DEC_STRIP / RPP;      // chunks a row, rows a pass
        const int chunk = lane % CH, sub = lane / CH;
        int seg = 0, n = 0, cols_phase = 0;
        bool go = busy, ok = true;
        // What the warp carries for head `cur`: a lane one column of every 32 of y, the column 16 b4 + 8 b3 + b2 + 2 (b1 b0)
        // of its bits (the order in which the collapse leaves them).
        const int my_col = (lane & 16) + (lane & 8) + ((lane >> 2) & 1) + 2 * (lane & 3);
        int cur = -1;
        float cm = -INFINITY, cl = 0.f, cy[COLS];
        // A strip's place in a tile: query head g of the key head, its first key, how many keys it holds; and the lane's
        // own row of it in the pools (a row on no valid page reads row 0 and is reported).
        int g = 0, valid = 0, row = 0;
        auto look = [&](const Walk<MASS>& at) {
            const Block& k = at.block;
            const int strip = (at.tile - k.tile0) * DEC_TILE_STRIPS + warp, j0 = (strip >> k.log_heads) * DEC_STRIP;
            g = k.g0 + (strip & ((1 << k.log_heads) - 1));
            valid = max(0, min(DEC_STRIP, at.s.seen - j0));
            row = 0;
            if (lane < valid) {
                row = p.pages.row(at.b, slot_of(p, at.s, j0 + lane));
                if (row < 0) { report(p.status, ST_PAGE); row = 0; }
            }
        };
        auto flush = [&]() {
            if (cur < 0) return;
            float* out = p.part + (static_cast<long long>(cur) + blockIdx.x) * DEC_TILE_STRIPS * REC + warp * REC;
#pragma unroll
            for (int c = 0; c < COLS; ++c) out[c * 32 + my_col] = cy[c];
            if (lane == 0) { out[D] = cm; out[D + 1] = cl; }
        };
        // The strip's 32 rows of a pool, coalesced, to the warp's own rows of one of the half's operand tiles.  Both tiles
        // are free between a segment's last score product and the next segment's first: Vr waits in the value tile for
        // the collapse, the next segment's R in the residual tile for the build, which replaces it in place.
        const uint32_t tiles_at = smem_u32(tile_hi);
        auto fetch = [&](const __nv_bfloat16* pool, const Walk<MASS>& at, uint32_t tile, int from_row) {
            const char* src = reinterpret_cast<const char*>(pool + static_cast<size_t>(at.head) * D + chunk * 8);
            const uint32_t pitch = static_cast<uint32_t>(p.Hkv) * D * 2;
            // rows of a batch first, then its copies: a shuffle's result is not waited for before every copy.  A row behind
            // the last key repeats row 0's place of the lane's shuffle; the build and the collapse leave it out.
            constexpr int BATCH = 8;
            const uint32_t at0 = tile + sw128_offset<128>(wq * 32 + sub, chunk);
#pragma unroll 1
            for (int i0 = 0; i0 < PASSES; i0 += BATCH) {
                uint32_t from[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) from[i] = __shfl_sync(0xFFFFFFFFu, from_row, (i0 + i) * RPP + sub);
#pragma unroll
                for (int i = 0; i < BATCH; ++i)            // RPP rows further on: the swizzle's row bits come round every 8 rows
                    copy16(RPP * (i0 + i) % 8 == 0 ? at0 + RPP * (i0 + i) * 128 : tile + sw128_offset<128>(wq * 32 + (i0 + i) * RPP + sub, chunk),
                           src + static_cast<uint64_t>(from[i]) * pitch);
            }
            copy_commit();
        };
        uint4 q = make_uint4(0, 0, 0, 0);
        auto prepare = [&](const Walk<MASS>& at) {
            look(at);
            if (valid > 0) fetch(p.R, at, tiles_at + L::TILE, row);
            else copy_commit();
            q = *reinterpret_cast<const uint4*>(p.Q + (static_cast<size_t>(at.b) * p.Hq + at.head * p.G + g) * D + chunk * 8);
        };
        while (go && !w.live(half)) go = w.next(p);
        if (go) prepare(w);
#pragma unroll 1
        while (go && ok) {
            // ---- operand tiles: value and residual of q o R
            copy_wait<0>();
            __syncwarp();
            auto build = [&](int i, bool all) {
                const int in = i * RPP + sub;
                const uint32_t at = sw128_offset<128>(wq * 32 + in, chunk);
                const uint4 r = *reinterpret_cast<const uint4*>(tile_hi + L::TILE + at);
                uint4 hi, lo;
                hi.x = mul_bf16x2(q.x, r.x); hi.y = mul_bf16x2(q.y, r.y);
                hi.z = mul_bf16x2(q.z, r.z); hi.w = mul_bf16x2(q.w, r.w);
                lo.x = residual_bf16x2(q.x, r.x, hi.x); lo.y = residual_bf16x2(q.y, r.y, hi.y);
                lo.z = residual_bf16x2(q.z, r.z, hi.z); lo.w = residual_bf16x2(q.w, r.w, hi.w);
                if (!all && in >= valid) hi = lo = make_uint4(0, 0, 0, 0);         // rows behind the last key
                st_shared_v4(tile_hi + at, hi.x, hi.y, hi.z, hi.w);
                st_shared_v4(tile_hi + L::TILE + at, lo.x, lo.y, lo.z, lo.w);
            };
            if (valid == DEC_STRIP) {
#pragma unroll 8
                for (int i = 0; i < PASSES; ++i) build(i, true);
            } else {
#pragma unroll 1
                for (int i = 0; i < PASSES; ++i) build(i, false);
            }
            fence_async_smem();
            warp_arrive(&bars[DB_A_FULL0 + half], lane);

            // ---- key steps
            float ref = 0.f, sum = 0.f;                    // reference maximum (scaled, base 2) of the strip; this row's sum
#pragma unroll 1
            for (int k = w.k0; k < w.k1; ++k, ++n) {
                ok = pipe_wait(&bars[DB_S_FULL0 + half], n & 1, fail, 2);
                if (!ok) break;
                tc_fence_after();
                if (k + 1 == w.k1) {                       // the tiles' last reader is done
                    if (valid > 0) fetch(p.Vr, w, tiles_at, row);
                    else copy_commit();
                }
                float col[4] = {0.f, 0.f, 0.f, 0.f};       // with masses: this warp's sums of columns c * 32 + lane
                // Raises the strip's reference to the maximum over its rows if a row exceeds it by 2^8; what was summed so
                // far follows.  (The products issued so far are complete: this step's scores came after them.)
                auto renew = [&](float mx) {
                    mx = lane < valid ? mx * p.c2 : -INFINITY;
                    if (k == w.k0) ref = fmaxf(warp_max(mx), -3e38f);      // scores that are -inf throughout count nothing, not NaN
                    else if (__any_sync(0xFFFFFFFFu, mx > ref + GROW)) {
                        const float now = warp_max(mx), f = fast_exp2(ref - now);
                        ref = now;
                        sum *= f;
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(tO + c * 16, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st16(tO + c * 16, o);
                        }
                    }
                };
                const uint64_t scale = pair_f32(p.c2, p.c2);
                const int cols = w.s.seen - k * DEC_KEYS, chunks = w.template chunks<WIDE>(k);          // visible columns of this step
                // Exponentials of 32 scores relative to the reference: their sum, their BF16 pairs to tensor memory (P of
                // chunk c covers score columns 16 c .. 16 c + 15, which are read by then), with masses the column sums.
                // Rows behind the last key contribute nothing: their exponent is -inf throughout.
                uint64_t s0 = pair_f32(0.f, 0.f), s1 = s0;
                auto exponentials = [&](const uint32_t (&x)[32], int c) {
                    const float shift1 = lane < valid ? -ref : -INFINITY;
                    const uint64_t shift = pair_f32(shift1, shift1);
                    float v[32];
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float a, b;
                        unpair_f32(fma_f32x2(pair_b32(x[i], x[i + 1]), scale, shift), a, b);
                        v[i] = fast_exp2(a);
                        v[i + 1] = fast_exp2(b);
                        if (i & 2) s1 = add_f32x2(s1, pair_f32(v[i], v[i + 1]));
                        else s0 = add_f32x2(s0, pair_f32(v[i], v[i + 1]));
                        packed[i / 2] = pack_bf16x2(v[i], v[i + 1]);
                    }
                    tmem_st16(tS + c * 16, packed);
                    if (MASS) {
                        const float t = sgring::warp_transpose_sum(v, lane);
                        col[0] = c == 0 ? t : col[0]; col[1] = c == 1 ? t : col[1];
                        col[2] = c == 2 ? t : col[2]; col[3] = c == 3 ? t : col[3];
                    }
                };
                // Two passes over the scores, the maximum and the exponentials, 64 columns at a time (the last step: 32), the
                // scores read twice from tensor memory: with all 128 of them in registers and everything unrolled the code
                // spills and outgrows the instruction cache, which holds all roles' code; with 32 at a time throughout, a
                // step takes 2950 cycles.
                // The 2 `pairs` first chunks have no hidden column.
                auto passes = [&](int pairs, int all) {
                    auto load = [&](int c, uint32_t (&x)[32]) {
                        tmem_ld32(tS + c * 32, x);
                        tmem_wait_ld();
                        if (c * 32 + 32 > cols) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[i] = c * 32 + i < cols ? x[i] : 0xFF800000u;          // -inf
                        }
                    };
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 2 * pairs; c += 2) {
                        uint32_t x[2][32];
                        tmem_ld32(tS + c * 32, x[0]);
                        tmem_ld32(tS + c * 32 + 32, x[1]);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fmaxf(__uint_as_float(x[0][i]), __uint_as_float(x[1][i])));
                    }
#pragma unroll 1
                    for (int c = 2 * pairs; c < all; ++c) {
                        uint32_t x[32];
                        load(c, x);
#pragma unroll
                        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(x[i]));
                    }
                    renew(mx);
#pragma unroll 1
                    for (int c = 0; c < 2 * pairs; c += 2) {
                        uint32_t x[2][32];
                        tmem_ld32(tS + c * 32, x[0]);
                        tmem_ld32(tS + c * 32 + 32, x[1]);
                        tmem_wait_ld();
                        exponentials(x[0], c);
                        exponentials(x[1], c + 1);
                    }
#pragma unroll 1
                    for (int c = 2 * pairs; c < all; ++c) {
                        uint32_t x[32];
                        load(c, x);
                        exponentials(x, c);
                    }
                };
                if (valid > 0) {
                    if (WIDE) passes((cols >= chunks * 32 ? chunks : chunks - 1) >> 1, chunks);
                    else if (cols >= DEC_KEYS) passes(2, 4);
                    else passes(0, chunks);
                }
                if (valid > 0) {
                    tmem_wait_st();
                    float a, b;
                    unpair_f32(add_f32x2(s0, s1), a, b);
                    sum += a + b;
                }
                tc_fence_before();
                warp_arrive(&bars[DB_P_FULL0 + half], lane);
                if (MASS && p.brief) {
                    const size_t at = (static_cast<size_t>(w.unit) + (k - w.k0)) * DEC_TILE_STRIPS + warp;
                    if (valid > 0) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) p.cols[at * 128 + c * 32 + lane] = col[c];
                        if (lane == 0) p.col_ref[at] = ref;
                    }
                } else if (MASS) {
                    // The half's column sums, relative to the largest of its four maxima: warps 2 and 3 hand theirs to
                    // 0 and 1, then 1 to 0.  (The first warp of a live half has keys, so that maximum is finite.)  Warp 0 adds
                    // them to what the CTA's earlier tiles of the head left, which is on its way meanwhile.
                    const size_t at = ((static_cast<size_t>(w.b * p.Hq + w.head * p.G + g) + blockIdx.x) * 2 + half) * p.col_steps + k;
                    const bool more = wq == 0 && w.again(k);
                    float old[4] = {0.f, 0.f, 0.f, 0.f}, old_ref = -INFINITY;
                    if (more) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) old[c] = p.cols[at * 128 + c * 32 + lane];
                        old_ref = p.col_ref[at];
                    }
                    float* buf = reinterpret_cast<float*>(smem + L::OFF_COL) + half * 256;
                    if (lane == 0) sh_ref[half * 4 + wq] = valid > 0 ? ref : -INFINITY;
                    if (wq >= 2) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) buf[(wq - 2) * 128 + c * 32 + lane] = col[c];
                    }
                    warp_arrive(&bars[DB_COL0 + half], lane);
                    ok = pipe_wait(&bars[DB_COL0 + half], cols_phase++ & 1, fail, 11);
                    if (!ok) break;
                    const float* rf = sh_ref + half * 4;
                    const float top = fmaxf(fmaxf(rf[0], rf[1]), fmaxf(rf[2], rf[3]));
                    if (wq < 2) {
                        const float f0 = fast_exp2(rf[wq] - top), f1 = fast_exp2(rf[wq + 2] - top);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            col[c] = col[c] * f0 + buf[wq * 128 + c * 32 + lane] * f1;
                            if (wq == 1) buf[128 + c * 32 + lane] = col[c];
                        }
                    }
                    warp_arrive(&bars[DB_COL0 + half], lane);
                    ok = pipe_wait(&bars[DB_COL0 + half], cols_phase++ & 1, fail, 11);
                    if (!ok) break;
                    if (wq == 0) {
                        const float joint = fmaxf(top, old_ref), f = fast_exp2(top - joint), f_old = fast_exp2(old_ref - joint);
#pragma unroll
                        for (int c = 0; c < 4; ++c) p.cols[at * 128 + c * 32 + lane] = (col[c] + buf[128 + c * 32 + lane]) * f + old[c] * f_old;
                        if (lane == 0) p.col_ref[at] = joint;          // the arrival below orders it before the warp's next look at it
                    }
                    warp_arrive(&bars[DB_COL0 + half], lane);
                    ok = pipe_wait(&bars[DB_COL0 + half], cols_phase++ & 1, fail, 11);
                    if (!ok) break;
                }
            }
            if (!ok) break;

            // ---- collapse: y = sum over the strip's rows of Vr o U.  The rows of Vr and the next strip's place are
            // fetched while the products finish.
            const int head = w.b * p.Hq + w.head * p.G + g, valid_now = valid;
            const int rec = w.slot * DEC_TILE_STRIPS + warp;
            do go = w.next(p); while (go && !w.live(half));
            if (go) prepare(w);
            else copy_commit();                            // an empty group: Vr is the last but one either way
            copy_wait<1>();
            __syncwarp();
            ok = pipe_wait(&bars[DB_O_DONE0 + half], seg & 1, fail, 3);
            if (!ok) break;
            tc_fence_after();
            if (valid_now > 0) {
                float l = lane < valid_now ? sum : 0.f;
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
                if (head != cur) {
                    flush();
                    cur = head;
                    cm = ref;
                    cl = 0.f;
#pragma unroll
                    for (int c = 0; c < COLS; ++c) cy[c] = 0.f;
                }
                const float m = fmaxf(cm, ref), f0 = fast_exp2(cm - m), f1 = fast_exp2(ref - m);
                cm = m;
                cl = cl * f0 + l * f1;
                // Lane L holds rows L/4 + 8 i and columns 8 k + 2 (L % 4), + 1 of 32 columns: four rows are added in the lane,
                // the eight lanes of a column pair by an exchange of halves, after which lane L has column L of the 32.
#pragma unroll 1
                for (int c = 0; c < COLS; ++c) {           // kept as a loop: the instruction cache holds all roles' code
                    uint32_t o[2][16];
                    tmem_ld_16x256b_x4(tO + c * 32, o[0]);
                    tmem_ld_16x256b_x4(tO + (16u << 16) + c * 32, o[1]);
                    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    // the row's swizzle is the lane's own: rows eight apart share it
                    const int r7 = (lane >> 2) & 7;
                    const uint8_t* rows = tile_hi + (wq * 32 + (lane >> 2)) * 128 + (c >> 1) * 128 * 128 + (lane & 3) * 4;
                    uint32_t u[4][4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint8_t* piece = rows + ((((c & 1) * 4 + k) ^ r7) << 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) u[i][k] = *reinterpret_cast<const uint32_t*>(piece + i * 1024);
                    }
                    tmem_wait_ld();
                    if (valid_now < DEC_STRIP) {           // rows behind the last key
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((lane >> 2) + 8 * i >= valid_now) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) u[i][k] = o[i >> 1][k * 4 + (i & 1) * 2] = o[i >> 1][k * 4 + (i & 1) * 2 + 1] = 0u;
                            }
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 f = unpack_bf16x2(u[i][k]);
                            v[2 * k] += f.x * __uint_as_float(o[i >> 1][k * 4 + (i & 1) * 2]);
                            v[2 * k + 1] += f.y * __uint_as_float(o[i >> 1][k * 4 + (i & 1) * 2 + 1]);
                        }
                    // v[2 k + e]: column 8 k + 2 (lane % 4) + e.  Bits 4, 3, 2 of the lane choose k's bits and e.
#pragma unroll
                    for (int st = 0; st < 3; ++st) {
                        const int o2 = 16 >> st, keep_n = 4 >> st;
                        const bool up = (lane & o2) != 0;
#pragma unroll
                        for (int k = 0; k < keep_n; ++k) {
                            const float send = up ? v[k] : v[k + keep_n], mine = up ? v[k + keep_n] : v[k];
                            v[k] = mine + __shfl_xor_sync(0xFFFFFFFFu, send, o2);
                        }
                    }
                    const float y = v[0] * f1;
#pragma unroll
                    for (int q = 0; q < COLS; ++q) cy[q] = q == c ? cy[q] * f0 + y : cy[q];
                }
                if (MASS) {
                    p.rows[static_cast<size_t>(rec) * DEC_STRIP + lane] = lane < valid_now ? sum : 0.f;
                    if (lane == 0) p.row_ref[rec] = ref;
                }
            }
            tc_fence_before();
            ++seg;
        }
        copy_wait<0>();
        flush();
    } else {
        sgring::reg_dec<88>();
        // the ring's stages: rows of a tile of S or Vs, 64 columns after the other
        constexpr int block_bytes = (WIDE ? DEC_WIDE : DEC_KEYS) * 128, stage_bytes = block_bytes * (D / 64);
        constexpr int stages = L::STAGES * L::TILE / stage_bytes;
        if (warp == 8 && busy) {
            // ================================================================== products
            const uint32_t issuer = elect_one();
            const uint32_t idesc_u = make_idesc_bf16(128, D, 0, 1);
            int n[2] = {0, 0}, seg[2] = {0, 0};            // steps and segments so far, per half
            int fill = 0;                                  // stages consumed
            bool go = true, ok = true;
            auto stage_desc = [&](int f, bool mn) {
                return make_smem_desc(smem_u32(smem + L::OFF_KV + (f % stages) * stage_bytes), mn ? block_bytes : 16, 1024, SWIZZLE_128B);
            };
            auto stage_wait = [&](int f) { return pipe_wait(&bars[DB_KV_FULL0 + f % stages], (f / stages) & 1, fail, 4); };
            auto scores = [&](int t, int f, int chunks) {
                const uint32_t idesc_x = make_idesc_bf16(128, chunks * 32, 0, 0);
                const uint64_t b = stage_desc(f, false);
                const uint32_t tX = tmem + t * 256;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const uint64_t a = make_smem_desc(smem_u32(smem + L::OFF_A + (2 * t + part) * L::TILE), 16, 1024, SWIZZLE_128B);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (kk & 3) * 32 / 16;
                        umma_ss_pred(tX, a + off + (kk >> 2) * (128 * 128 / 16), b + off + (kk >> 2) * (block_bytes / 16), idesc_x, part > 0 || kk > 0,
                                     issuer);
                    }
                }
                umma_commit_pred(&bars[DB_S_FULL0 + t], issuer);
            };
#pragma unroll 1
            while (go && ok) {
                const bool two = w.live(1);
                ok = stage_wait(fill);
                for (int t = 0; t < (two ? 2 : 1) && ok; ++t) {
                    ok = pipe_wait(&bars[DB_A_FULL0 + t], seg[t] & 1, fail, 5);
                    if (!ok) break;
                    tc_fence_after();
                    scores(t, fill, w.template chunks<WIDE>(w.k0));
                }
                if (!ok) break;
                umma_commit_pred(&bars[DB_KV_EMPTY0 + fill % stages], issuer);
#pragma unroll 1
                for (int k = w.k0; k < w.k1 && ok; ++k) {
                    const bool more = k + 1 < w.k1;
                    const int chunks = w.template chunks<WIDE>(k);
                    ok = stage_wait(fill + 1);
                    for (int t = 0; t < (two ? 2 : 1) && ok; ++t) {
                        ok = pipe_wait(&bars[DB_P_FULL0 + t], n[t] & 1, fail, 6);
                        if (!ok) break;
                        ++n[t];
                        tc_fence_after();
                        const uint64_t b = stage_desc(fill + 1, true);
                        auto product = [&](int kk) {
                            umma_ts_pred(tmem + t * 256 + 128, tmem + t * 256 + kk * 8, b + kk * (2048 / 16), idesc_u, k > w.k0 || kk > 0, issuer);
                        };
                        if (chunks == 4) {
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk) product(kk);
                        } else {
#pragma unroll 1
                            for (int kk = 0; kk < 2 * chunks; ++kk) product(kk);
                        }
                        if (!more) umma_commit_pred(&bars[DB_O_DONE0 + t], issuer);
                        else {
                            if (t == 0) ok = stage_wait(fill + 2);
                            if (!ok) break;
                            scores(t, fill + 2, w.template chunks<WIDE>(k + 1));
                        }
                    }
                    if (!ok) break;
                    umma_commit_pred(&bars[DB_KV_EMPTY0 + (fill + 1) % stages], issuer);
                    if (more) umma_commit_pred(&bars[DB_KV_EMPTY0 + (fill + 2) % stages], issuer);
                    fill += 2;
                }
                ++seg[0];
                if (two) ++seg[1];
                go = w.next(p);
            }
            // nothing of this warp's is in flight when the tensor memory is given back
            umma_commit_pred(&bars[DB_DRAIN], issuer);
            pipe_wait(&bars[DB_DRAIN], 0, fail, 7);
        } else if (warp >= 9 && busy) {
            // ================================================================== rows of S and Vs
            const int mine = lane * DEC_COPY_WARPS + warp - 9;         // this lane's box, or group of four rows
            int fill = 0;
            bool go = true, ok = true;
#pragma unroll 1
            while (go && ok) {
#pragma unroll 1
                for (int k = w.k0; k < w.k1 && ok; ++k) {
                    const bool boxes = !WIDE && p.box > 0 && (k + 1) * DEC_KEYS <= w.s.seen;
                    const int rows = boxes ? p.box : 4;
                    const int wanted = w.template chunks<WIDE>(k) * 32;
                    const bool any = mine * rows < wanted;
                    int row[4] = {0, 0, 0, 0};
                    if (any) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (i > 0 && boxes) break;
                            // columns behind the last key repeat its row: they are masked, and a finite row stays finite
                            const int e = min(k * DEC_KEYS + mine * rows + i, w.s.seen - 1);
                            row[i] = p.pages.row(w.b, slot_of(p, w.s, e));
                            if (row[i] < 0) { report(p.status, ST_PAGE); row[i] = 0; }
                        }
                    }
#pragma unroll 1
                    for (int kind = 0; kind < 2; ++kind, ++fill) {
                        const int st = fill % stages;
                        uint64_t* full = &bars[DB_KV_FULL0 + st];
                        if (fill >= stages) ok = pipe_wait(&bars[DB_KV_EMPTY0 + st], (fill / stages - 1) & 1, fail, 8);
                        if (!ok) break;
                        // One arrival of every copy warp, the one of warp 9 names the bytes; other warps' bytes may come before
                        // it.  A warp without a box of its own (boxes of 64 rows and more) arrives too: a stage that went
                        // round twice while it waits for the first would look to it as if it had not gone round at all.
                        if (lane == 0) {
                            if (warp == 9) mbar_arrive_expect_tx(full, wanted * D * 2);
                            else mbar_arrive(full);
                        }
                        __syncwarp();
                        if (any) {
                            uint8_t* dst = smem + L::OFF_KV + st * stage_bytes + mine * rows * 128;
#pragma unroll
                            for (int h = 0; h < D / 64; ++h) {
                                const int x = w.head * D + h * 64;
                                if (boxes) tma_load_2d(dst + h * block_bytes, kind ? &p.tmVs_box : &p.tmS_box, x, row[0], full);
                                else tma_gather4(dst + h * block_bytes, kind ? &p.tmVs : &p.tmS, x, row, full);
                            }
                        }
                        __syncwarp();
                    }
                }
                go = go && w.next(p);
            }
            // every copy that was asked for has landed before the CTA ends
            for (int f = max(0, fill - stages); f < fill; ++f)
                pipe_wait(&bars[DB_KV_FULL0 + f % stages], (f / stages) & 1, fail, 9);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, 512);
    if (tid == 0 && *fail) report(p.status, *fail & 0xFF);
}

// The partials of one head, shared out over eight warps and added in a fixed order; a warp's lanes take the columns.
template <int D, bool MASS>
__global__ void __launch_bounds__(256) decode_join_kernel(const __grid_constant__ DecodeParams p, int ctas) {
    constexpr int REC = D + 4, COLS = D / 32;
    __shared__ float sh_m[8], sh_l[8], sh_y[8][D];
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq, kv = hq / p.G, g = hq % p.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_previous_kernel();
    const Shape s = shape_of<MASS>(p, b);
    __nv_bfloat16* y = p.Y + static_cast<size_t>(blockIdx.x) * D;
    if (s.seen == 0) {
        if (threadIdx.x < D) y[threadIdx.x] = __float2bfloat16_rn(0.f);
        return;
    }
    const int total = p.unit_base[p.B], units0 = p.unit_base[b] + kv * s.tiles * s.steps;
    const Block k = block_of_head<MASS>(p, s, g);
    const int u0 = units0 + k.tile0 * s.steps, u1 = u0 + block_tiles(1 << k.log_heads, s.groups) * s.steps;
    const int c0 = cta_of(u0, total, ctas), c1 = cta_of(u1 - 1, total, ctas);
    // records: of every CTA on the head's tiles, those of the 8 / heads warps that had its strips; shared out over the warps
    const int log_warps = 3 - k.log_heads, records = (c1 - c0 + 1) << log_warps;
    float m = -INFINITY, l = 0.f, acc[COLS];
#pragma unroll
    for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int i = warp; i < records; i += 8) {
        const int c = c0 + (i >> log_warps), from_warp = ((i & ((1 << log_warps) - 1)) << k.log_heads) + g - k.g0;
        // the first of the head's tiles that CTA c went through, and whether it had keys for that warp
        const int from = max(stretch(total, c, ctas), u0), to = min(stretch(total, c + 1, ctas), u1);
        if (from >= to) continue;
        const int strip = (from - u0) / s.steps * DEC_TILE_STRIPS + from_warp;
        if (strip >> k.log_heads >= s.groups) continue;
        const float* r = p.part + (static_cast<long long>(blockIdx.x) + c) * DEC_TILE_STRIPS * REC + from_warp * REC;
        const float rm = r[D], top = fmaxf(m, rm), f0 = m > -INFINITY ? fast_exp2(m - top) : 0.f, f1 = fast_exp2(rm - top);
        m = top;
        l = l * f0 + r[D + 1] * f1;
#pragma unroll
        for (int q = 0; q < COLS; ++q) acc[q] = acc[q] * f0 + r[q * 32 + lane] * f1;
    }
    if (lane == 0) { sh_m[warp] = m; sh_l[warp] = l; }            // a warp without records leaves -inf, 0 and zeros
#pragma unroll
    for (int q = 0; q < COLS; ++q) sh_y[warp][q * 32 + lane] = acc[q];
    __syncthreads();
    if (threadIdx.x < D) {
        float top = sh_m[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, sh_m[i]);
        float a = 0.f, ls = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = fast_exp2(sh_m[i] - top);
            a += sh_y[i][threadIdx.x] * f;
            ls += sh_l[i] * f;
        }
        y[threadIdx.x] = __float2bfloat16_rn(a / ls);
        if (MASS && threadIdx.x == 0) p.lse[blockIdx.x] = top + log2f(ls);
    }
}

// Adds every visible slot's share of the attention to its mass: up to four threads a slot, which share the heads; heads and
// partials in a fixed order.
constexpr int MASS_PARTS = 4;
__global__ void __launch_bounds__(128 * MASS_PARTS) decode_mass_kernel(const __grid_constant__ DecodeParams p, int ctas) {
    __shared__ float sums[MASS_PARTS][128];
    const int b = blockIdx.y / p.Hkv, kv = blockIdx.y % p.Hkv;
    wait_for_previous_kernel();
    const Shape s = shape_of<true>(p, b);
    const int e = blockIdx.x * 128 + threadIdx.x;
    if (blockIdx.x * 128 >= static_cast<unsigned>(s.seen)) return;
    const int row = e < s.seen ? p.pages.row(b, slot_of(p, s, e)) : -1;
    const int total = p.unit_base[p.B], units0 = p.unit_base[b] + kv * s.tiles * s.steps;
    const int tiles0 = p.tile_base[b] + kv * s.tiles;
    const int step = e / DEC_KEYS, col = e % DEC_KEYS;
    float share = 0.f;
    for (int g = threadIdx.y; row >= 0 && g < p.G; g += blockDim.y) {
        const float lse = p.lse[b * p.Hq + kv * p.G + g];
        const Block k = block_of_head<true>(p, s, g);
        auto strip_of = [&](int group) { return (group << k.log_heads) + g - k.g0; };
        // as j: the row's sums, of every CTA that took a part of the tile's keys
        const int mine = strip_of(e / DEC_STRIP), tile = k.tile0 + mine / DEC_TILE_STRIPS;
        const int u = units0 + tile * s.steps;
        const int c0 = cta_of(u, total, ctas), c1 = cta_of(u + s.steps - 1, total, ctas);
        for (int c = c0; c <= c1; ++c) {
            if (stretch(total, c, ctas) >= stretch(total, c + 1, ctas)) continue;
            const size_t rec = static_cast<size_t>(tiles0 + tile + c) * DEC_TILE_STRIPS + mine % DEC_TILE_STRIPS;
            share += p.rows[rec * DEC_STRIP + e % DEC_STRIP] * fast_exp2(p.row_ref[rec] - lse);
        }
        // as k: the column's sums over the head's rows
        if (p.brief) {
#pragma unroll 4
            for (int group = 0; group < s.groups; ++group) {
                const int strip = strip_of(group);
                const size_t at = (static_cast<size_t>(units0) + k.tile0 + strip / DEC_TILE_STRIPS) * DEC_TILE_STRIPS + strip % DEC_TILE_STRIPS;
                share += p.cols[at * 128 + col] * fast_exp2(p.col_ref[at] - lse);
            }
        } else {
            // of every CTA that came by this key step, the half tile of its second half if it saw one
            const int u0 = units0 + k.tile0 * s.steps, u1 = u0 + block_tiles(1, s.groups) * s.steps;
            const int first = cta_of(u0, total, ctas), last = cta_of(u1 - 1, total, ctas);
            // no branches: the loads of several CTAs are under way together
#pragma unroll 4
            for (int c = first; c <= last; ++c) {
                const int from = max(stretch(total, c, ctas), u0) - u0, to = min(stretch(total, c + 1, ctas), u1) - u0;
                const int t = from / s.steps + (step < from % s.steps ? 1 : 0);        // its first tile with the step
                const bool one = t * s.steps + step < to, two = one && t * 256 + 128 < s.seen;
                const size_t at = (static_cast<size_t>(b * p.Hq + kv * p.G + g) + c) * 2 * p.col_steps + step, at2 = at + p.col_steps;
                const float v1 = one ? p.cols[at * 128 + col] : 0.f, r1 = one ? p.col_ref[at] : -INFINITY;
                const float v2 = two ? p.cols[at2 * 128 + col] : 0.f, r2 = two ? p.col_ref[at2] : -INFINITY;
                share += v1 * fast_exp2(r1 - lse);
                share += v2 * fast_exp2(r2 - lse);
            }
        }
    }
    sums[threadIdx.y][threadIdx.x] = share;
    __syncthreads();
    if (threadIdx.y > 0 || row < 0) return;
    for (unsigned i = 1; i < blockDim.y; ++i) share += sums[i][threadIdx.x];
    // atomically: sequences may share the pages of a prefix, and each adds its own share (elsewhere there is one addition)
    atomicAdd(p.mass + static_cast<long long>(row) * p.Hkv + kv, share / (2.f * p.G));
}

}  // namespace serve
