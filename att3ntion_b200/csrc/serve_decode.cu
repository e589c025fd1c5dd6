// C-ABI entry points of the single-token gather over a paged cache: argument checks, workspace layout, launches.
#include <algorithm>
#include <cmath>

#include "serve_decode.cuh"

namespace {

struct Layout {
    size_t part, rows, row_ref, cols, col_ref, lse, unit_base, tile_base, bytes;
    long long units;
    int ctas, wide, brief, col_steps;
};

// The workspace for the longest sequences that the arguments admit.
Layout layout(int B, int Hq, int Hkv, int D, int window, int sinks, long long max_slots, bool mass) {
    Layout o = {};
    const long long seen = window > 0 ? std::min<long long>(max_slots, static_cast<long long>(window) + sinks) : max_slots;
    const long long G = Hq / Hkv;
    const long long groups = (seen + 31) / 32;
    auto block = [&](long long heads) { return (heads * groups + 7) / 8; };          // tiles of a block of heads
    o.brief = mass && seen <= serve::DEC_KEYS;
    const long long per_key_head = mass && !o.brief ? G * block(1) : G / 8 * groups + (G & 4 ? block(4) : 0) + (G & 2 ? block(2) : 0) + (G & 1 ? block(1) : 0);
    const long long tiles = static_cast<long long>(B) * Hkv * per_key_head;
    // One step of up to 192 keys a tile in place of two, where the longest needs no more (128 sequences of 8 heads at
    // window 128 with 4 sinks: 45 us in place of 58).  The masses' column sums are laid out for steps of 128.
    o.wide = !mass && seen > serve::DEC_KEYS && seen <= serve::DEC_WIDE;
    o.units = tiles * (o.wide ? 1 : (seen + 127) / 128);
    o.ctas = static_cast<int>(std::max<long long>(1, std::min<long long>(att3::sm_count(), o.units)));
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
    o.part = take((static_cast<size_t>(B) * Hq + o.ctas) * 8 * (D + 4) * 4);
    o.unit_base = take((static_cast<size_t>(B) + 1) * 4);
    o.tile_base = take((static_cast<size_t>(B) + 1) * 4);
    if (mass) {
        o.rows = take((static_cast<size_t>(tiles) + o.ctas) * 8 * 32 * 4);
        o.row_ref = take((static_cast<size_t>(tiles) + o.ctas) * 8 * 4);
        // column sums by (head, CTA): no more pairs than heads and CTAs, since both only go up along the line of units
        o.col_steps = static_cast<int>((seen + 127) / 128);
        const size_t sums = o.brief ? static_cast<size_t>(o.units) * 8 : (static_cast<size_t>(B) * Hq + o.ctas) * 2 * o.col_steps;
        o.cols = take(sums * 128 * 4);
        o.col_ref = take(sums * 4);
        o.lse = take(static_cast<size_t>(B) * Hq * 4);
    }
    o.bytes = at;
    return o;
}

int check(const char* who, int B, int Hq, int Hkv, int D, int window, int sinks) {
    if (B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0)
        return att3::set_error(ATT3_ERR_INVALID, "%s: Hq=%d is not divisible by Hkv=%d", who, Hq, Hkv);
    if (D != 64 && D != 128) return att3::set_error(ATT3_ERR_INVALID, "%s: D must be 64 or 128, got %d", who, D);
    if (window < 0 || sinks < 0) return att3::set_error(ATT3_ERR_INVALID, "%s: window and sinks must not be negative", who);
    if (static_cast<long long>(B) * Hq >= (1 << 24) || static_cast<long long>(window) + sinks > (1 << 30))
        return att3::set_error(ATT3_ERR_INVALID, "%s: too many heads, or too wide a window", who);
    return ATT3_OK;
}

template <int D, bool MASS, bool WIDE>
int launch(const serve::DecodeParams& p, const Layout& lay, long long max_seen, cudaStream_t st, const char* who) {
    constexpr int smem = serve::DecSmem<D>::BYTES;
    cudaError_t e = cudaFuncSetAttribute(serve::decode_kernel<D, MASS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return att3::set_cuda_error(e, who);
    att3::count_launch(4, MASS ? 3 : 2);
    const att3::TimedLaunch timed(att3::K_SERVE, st);
    e = serve::launch_early(serve::decode_kernel<D, MASS, WIDE>, dim3(lay.ctas), dim3(serve::DEC_THREADS), smem, st, p);
    if (e == cudaSuccess) e = serve::launch_early(serve::decode_join_kernel<D, MASS>, dim3(p.B * p.Hq), dim3(256), 0, st, p, lay.ctas);
    if (MASS && e == cudaSuccess)
        e = serve::launch_early(serve::decode_mass_kernel, dim3(static_cast<unsigned>((max_seen + 127) / 128), p.B * p.Hkv), dim3(128, std::min(p.G, serve::MASS_PARTS)), 0, st, p, lay.ctas);
    return e == cudaSuccess ? ATT3_OK : att3::set_cuda_error(e, who);
}

}  // namespace

extern "C" size_t att3_sg_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int window, int sinks, int max_slots, int with_mass) {
    if (check("att3_sg_decode_workspace_bytes", B, Hq, Hkv, D, window, sinks) || max_slots < 1) return 0;
    return layout(B, Hq, Hkv, D, window, sinks, max_slots, with_mass != 0).bytes;
}

extern "C" int att3_sg_decode(const void* Q, const void* R, const void* S, const void* Vr, const void* Vs, float* mass, void* Y,
                              const att3_gather_pages* pages, const int32_t* lengths, int B, int Hq, int Hkv, int D, int window,
                              int sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "att3_sg_decode";
    if (int rc = check(who, B, Hq, Hkv, D, window, sinks)) return rc;
    if (B == 0) return ATT3_OK;
    if (int rc = att3::check_gather_pages(pages, who)) return rc;
    if (!Q || !R || !S || !Vr || !Vs || !Y || !lengths) return att3::set_error(ATT3_ERR_INVALID, "%s: null tensor", who);
    for (const void* q : {Q, R, S, Vr, Vs, static_cast<const void*>(Y)})
        if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return att3::set_error(ATT3_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
    const long long most = pages->per_sequence * pages->page_size;
    if (mass && static_cast<long long>(B) * Hkv > 65535)
        return att3::set_error(ATT3_ERR_INVALID, "%s: with masses at most 65535 sequences times key heads, got %lld", who, static_cast<long long>(B) * Hkv);
    const Layout lay = layout(B, Hq, Hkv, D, window, sinks, most, mass != nullptr);
    if (lay.units > 0x7FFFFFFFll)
        return att3::set_error(ATT3_ERR_INVALID, "%s: the table's width, sequences and heads admit more than 2^31 - 1 units of work", who);
    if (!workspace || workspace_bytes < lay.bytes || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return att3::set_error(ATT3_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed", who, lay.bytes);
    if (!att3::require_sm100(who)) return ATT3_ERR_UNSUPPORTED;
    serve::DecodeParams p = {};
    p.Q = static_cast<const __nv_bfloat16*>(Q);
    p.R = static_cast<const __nv_bfloat16*>(R);
    p.Vr = static_cast<const __nv_bfloat16*>(Vr);
    // boxes of the largest power of two that divides the page, from 8 rows on (below that a box saves nothing over a gather)
    p.box = static_cast<int>(std::min<int64_t>(pages->page_size & -pages->page_size, serve::DEC_KEYS));
    if (window > 0 || p.box < 8) p.box = 0;
    const size_t rows = static_cast<size_t>(pages->pages) * pages->page_size;
    if (int rc = att3::make_gather_tensor_map(&p.tmS, S, rows, Hkv * D, 1, who)) return rc;
    if (int rc = att3::make_gather_tensor_map(&p.tmVs, Vs, rows, Hkv * D, 1, who)) return rc;
    if (p.box) {
        if (int rc = att3::make_gather_tensor_map(&p.tmS_box, S, rows, Hkv * D, p.box, who)) return rc;
        if (int rc = att3::make_gather_tensor_map(&p.tmVs_box, Vs, rows, Hkv * D, p.box, who)) return rc;
    }
    p.Y = static_cast<__nv_bfloat16*>(Y);
    p.mass = mass;
    p.lengths = lengths;
    p.pages = serve::make_pages(pages->table, pages->table_stride, pages->per_sequence, pages->pages, pages->page_size);
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.window = window; p.sinks = sinks;
    p.wide = lay.wide;
    p.brief = lay.brief;
    p.col_steps = lay.col_steps;
    p.c2 = sgring::LOG2E / std::sqrt(static_cast<float>(D));
    char* ws = static_cast<char*>(workspace);
    p.part = reinterpret_cast<float*>(ws + lay.part);
    p.unit_base = reinterpret_cast<int*>(ws + lay.unit_base);
    p.tile_base = reinterpret_cast<int*>(ws + lay.tile_base);
    p.rows = reinterpret_cast<float*>(ws + lay.rows);
    p.row_ref = reinterpret_cast<float*>(ws + lay.row_ref);
    p.cols = reinterpret_cast<float*>(ws + lay.cols);
    p.col_ref = reinterpret_cast<float*>(ws + lay.col_ref);
    p.lse = reinterpret_cast<float*>(ws + lay.lse);
    if (!(p.status = att3::serve_status_ptr())) return att3::set_error(ATT3_ERR_CUDA, "%s: status word not resolvable", who);
    const long long seen = window > 0 ? std::min<long long>(most, static_cast<long long>(window) + sinks) : most;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (D == 128)
        return mass ? launch<128, true, false>(p, lay, seen, st, who)
                    : lay.wide ? launch<128, false, true>(p, lay, seen, st, who) : launch<128, false, false>(p, lay, seen, st, who);
    return mass ? launch<64, true, false>(p, lay, seen, st, who)
                : lay.wide ? launch<64, false, true>(p, lay, seen, st, who) : launch<64, false, false>(p, lay, seen, st, who);
}
