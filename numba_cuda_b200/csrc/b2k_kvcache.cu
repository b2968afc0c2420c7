// The quantised paged cache of keys and values: written as tokens arrive
// (b2k_cache_write), written straight from norm and rotation (b2k_norm_rotate_write),
// and read back by page table (b2k_cache_read).  The conversions are those of the
// reference's scalar intrinsics (numba/cuda/_internal/cuda_fp8.py:3341-3374) around a
// scale per head or per block of a head.
#include "b2k_heads_forward.cuh"

namespace {

using namespace headwise;

struct ReadSide {
    const uint8_t *codes;
    const void *scales;
    int64_t code_page, code_slot, code_head, scale_page, scale_slot, scale_head;
    void *out;
    int64_t out_token, out_head;
    int heads, dim, group;
};
struct ReadParams {
    ReadSide side[2];
    int64_t rows, pages, page_size;
    const void *table, *offsets;
    int64_t table_stride, table_width, seqs;
    int table_bytes, offset_bytes, e5m2, e8m0;
};

template <typename T> struct Largest;
template <> struct Largest<float> { static constexpr float value = FLT_MAX; };
template <> struct Largest<__half> { static constexpr float value = 65504.0f; };
template <> struct Largest<__nv_bfloat16> { static constexpr float value = 3.38953138925153547590470800371487866880e38f; };

__device__ __forceinline__ float decode(uint8_t code, int e5m2) {
    uint32_t two;
    if (e5m2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(two) : "h"(static_cast<uint16_t>(code)));
    else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"(static_cast<uint16_t>(code)));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(two)));
}
// A value beyond the output's range is its largest one; a NaN stays.
template <typename T>
__device__ __forceinline__ float saturated(float v) {
    return fabsf(v) > Largest<T>::value ? copysignf(Largest<T>::value, v) : v;
}

__device__ __forceinline__ float load_scale(const void *scales, int64_t at, int e8m0) {
    if (!e8m0) return static_cast<const float *>(scales)[at];
    const uint32_t e = static_cast<const uint8_t *>(scales)[at];
    // 2^(e - 127); code 0 is the subnormal 2^-127, 255 is NaN
    return __uint_as_float(e == 0 ? 0x00400000u : e == 255 ? 0x7FC00000u : e << 23);
}

// One warp per row of the output (a token of one side), lanes along its items.
template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
    const ReadSide &s = p.side[blockIdx.y];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32;
    if (row >= p.rows || s.heads == 0) return;
    const int64_t b = paging::sequence_of_row(p.offsets, p.offset_bytes, p.seqs, row);
    if (b < 0) return;
    const paging::Place at = paging::place_in_sequence(row - paging::load_index(p.offsets, p.offset_bytes, b),
                                                             p.table, p.table_stride, p.table_width, p.table_bytes, b,
                                                             p.pages, p.page_size);
    for (int head = 0; head < s.heads; ++head) {
        T *out = static_cast<T *>(s.out) + row * s.out_token + head * s.out_head;
        const uint8_t *codes = s.codes + at.page * s.code_page + at.slot * s.code_slot + head * s.code_head;
        const int64_t scales = at.page * s.scale_page + at.slot * s.scale_slot + head * s.scale_head;
        for (int d = threadIdx.x % 32; d < s.dim; d += 32) {
            float v = 0.0f;
            if (at.ok) v = saturated<T>(decode(codes[d], p.e5m2) * load_scale(s.scales, scales + d / s.group, p.e8m0));
            out[d] = Convert<T>::down(v);
        }
    }
}

int check_slots(const void *slots, int slot_bytes, int64_t tokens, const char *name) {
    return tokens ? check_indices(slots, slot_bytes, name, "slots") : B2K_OK;
}

}  // namespace

extern "C" {

int b2k_cache_write(const b2k_cache *cache, int format, int64_t tokens, const b2k_heads *k, const b2k_heads *v,
                    const void *slots_dev, int slot_bytes, void *stream) {
    B2K_RANGE("b2k_cache_write");
    const char *name = "b2k_cache_write";
    if (int rc = check_cache(cache, name)) return rc;
    if (int rc = check_tokens(format, tokens, name)) return rc;
    if (k == nullptr || v == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    if (int rc = check_slots(slots_dev, slot_bytes, tokens, name)) return rc;
    Params p{};
    const b2k_heads *in[2] = {k, v};
    const b2k_pages *side[2] = {&cache->k, &cache->v};
    for (int i = 0; i < 2; ++i) {
        const char *what = i ? "v" : "k";
        if (int rc = check_heads(*in[i], name, what, tokens, item_bytes(format), false)) return rc;
        if (int rc = check_side(*side[i], *in[i], *cache, name, what, true)) return rc;
        if (in[i]->heads == 0) continue;
        set_input(p.role[1 + i], *in[i], tokens);
        set_pages(p, p.role[1 + i], *cache, *side[i]);
    }
    if (tokens == 0 || cache->pages == 0) return B2K_OK;
    p.tokens = tokens;
    p.slots = slots_dev;
    p.slot_bytes = slot_bytes;
    const Plan plan = choose(p, format, nullptr);
    return launch_forward<kWrite>(p, format, plan, b2k::as_stream(stream), name);
}

int b2k_norm_rotate_write(const b2k_rotation *r, const b2k_heads *v, const b2k_heads *q_out, const b2k_cache *cache,
                          const void *slots_dev, int slot_bytes, void *stream) {
    B2K_RANGE("b2k_norm_rotate_write");
    const char *name = "b2k_norm_rotate_write";
    if (int rc = check_rotation(r, name)) return rc;
    if (int rc = check_cache(cache, name)) return rc;
    if (v == nullptr || q_out == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    const int itemsize = item_bytes(r->format);
    if (int rc = check_heads(*v, name, "v", r->tokens, itemsize, false)) return rc;
    if (int rc = check_heads(*q_out, name, "q_out", r->tokens, itemsize, true)) return rc;
    if (int rc = check_like(*q_out, r->q, name, "q_out")) return rc;
    if (int rc = check_side(cache->k, r->k, *cache, name, "k", true)) return rc;
    if (int rc = check_side(cache->v, *v, *cache, name, "v", true)) return rc;
    if (int rc = check_slots(slots_dev, slot_bytes, r->tokens, name)) return rc;
    if (r->tokens == 0) return B2K_OK;
    Params p{};
    if (r->q.heads) {
        set_input(p.role[0], r->q, r->tokens);
        set_output(p.role[0], *q_out, r->tokens);
    }
    if (r->k.heads) {
        set_input(p.role[1], r->k, r->tokens);
        set_pages(p, p.role[1], *cache, cache->k);
    }
    if (v->heads) {
        set_input(p.role[2], *v, r->tokens);
        set_pages(p, p.role[2], *cache, cache->v);
    }
    p.tokens = r->tokens;
    p.slots = slots_dev;
    p.slot_bytes = slot_bytes;
    set_rotation(p, *r);
    const Plan plan = choose(p, r->format, r);
    return launch_forward<kBoth>(p, r->format, plan, b2k::as_stream(stream), name);
}

int b2k_cache_read(const b2k_cache *cache, int format, int64_t rows, const b2k_heads *k_out, const b2k_heads *v_out,
                   const void *table_dev, int64_t table_stride, int64_t table_width, int table_bytes,
                   const void *offsets_dev, int64_t seqs, int offset_bytes, void *stream) {
    B2K_RANGE("b2k_cache_read");
    const char *name = "b2k_cache_read";
    if (int rc = check_cache(cache, name)) return rc;
    if (int rc = check_tokens(format, rows, name)) return rc;
    if (k_out == nullptr || v_out == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    if (seqs < 0 || table_width < 0) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: negative size of the page table", name);
    ReadParams p{};
    const b2k_heads *out[2] = {k_out, v_out};
    const b2k_pages *side[2] = {&cache->k, &cache->v};
    for (int i = 0; i < 2; ++i) {
        const char *what = i ? "v" : "k";
        if (int rc = check_heads(*out[i], name, i ? "v_out" : "k_out", rows, item_bytes(format), true)) return rc;
        if (int rc = check_side(*side[i], *out[i], *cache, name, what, false)) return rc;
        if (out[i]->heads == 0) continue;
        Params shape{};
        Role r{};
        set_output(r, *out[i], rows);
        r.heads = static_cast<int>(out[i]->heads);
        set_pages(shape, r, *cache, *side[i]);
        p.side[i] = ReadSide{r.codes, r.scales, r.code_page, r.code_slot, r.code_head, r.scale_page, r.scale_slot,
                             r.scale_head, r.out, r.out_token, r.out_head, r.heads, static_cast<int>(out[i]->dim),
                             r.group};
    }
    if (rows == 0 || seqs == 0 || (k_out->heads == 0 && v_out->heads == 0)) return B2K_OK;
    if (int rc = check_indices(offsets_dev, offset_bytes, name, "offsets")) return rc;
    if (table_width > 0)
        if (int rc = check_indices(table_dev, table_bytes, name, "the page table")) return rc;
    p.rows = rows;
    p.pages = cache->pages;
    p.page_size = cache->page_size;
    p.table = table_dev;
    p.offsets = offsets_dev;
    p.table_stride = table_stride;
    p.table_width = table_width;
    p.seqs = seqs;
    p.table_bytes = table_bytes;
    p.offset_bytes = offset_bytes;
    p.e5m2 = cache->code_format == B2K_FMT_E5M2;
    p.e8m0 = cache->scale_format == B2K_FMT_E8M0;
    const int64_t blocks = (rows + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > INT_MAX) return b2k::fail(B2K_ERR_TOO_LARGE, "%s: too many rows for one launch", name);
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    const cudaStream_t st = b2k::as_stream(stream);
    if (format == B2K_FMT_F32) cache_read_kernel<float><<<grid, kThreads, 0, st>>>(p);
    else if (format == B2K_FMT_F16) cache_read_kernel<__half><<<grid, kThreads, 0, st>>>(p);
    else cache_read_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    B2K_RETURN_IF_LAUNCH_FAILED(name);
    b2k::note_launch();
    return B2K_OK;
}

}  // extern "C"
