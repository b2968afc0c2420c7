// The quantised paged cache of keys and values: written as tokens arrive
// (b2k_cache_write), written straight from norm and rotation (b2k_norm_rotate_write),
// and read back by page table (b2k_cache_read).  The conversions are those of the
// reference's scalar intrinsics (numba/cuda/_internal/cuda_fp8.py:3341-3374) around a
// scale per head or per block of a head.
//
// Writing is the forward row kernel (b2k_heads_forward.cuh) with its store replaced: the
// group's largest magnitude by shuffles, the scale, the codes.  Measured: 32768 tokens x
// (8 + 8) heads of 128 bf16 items 40 to 42 us = 4.9 to 5.1 TB/s (issue slots 67% busy), about what a
// plain copy of those bytes takes; with norm, rotation and 64 query heads beside it, 8192
// tokens 63 us.
#include <algorithm>

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
    int tile;                       // output rows a block owns, at most kTileRows
};

// ---- reading back ---------------------------------------------------------------------
// A block owns a tile of consecutive output rows of one side.  Its first threads find
// each row's place (a binary search over the offsets, one page-table entry); then every
// thread keeps one chunk of CV items of a row and walks down the tile's rows with
// kReadRows loads in flight, so index arithmetic is paid once a thread.  HBM bounds it:
// one byte in, sizeof(T) bytes out per item.  65536 tokens x (8 + 8) heads of 128 items to
// bf16: 65 us = 6.3 TB/s (one warp a token and single items: 316 us).
constexpr int kTileRows = 32;
constexpr int kReadRows = 4;

// Exact: every E4M3 and E5M2 value is a float16.
template <int E5M2>
__device__ __forceinline__ float2 decode2(uint16_t two_codes) {
    uint32_t two;
    if constexpr (E5M2) asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(two) : "h"(two_codes));
    else asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"(two_codes));
    return __half22float2(*reinterpret_cast<const __half2 *>(&two));
}

// The one rounding of a value that is read: the float32 product of code and scale to the
// output's type.  A finite code can land beyond that type's range (65504 in float16 under
// a scale rounded up to a power of two reads back as 65536), so the store saturates.
// A NaN stays one.
__device__ __forceinline__ float saturated(float v) { return fabsf(v) > FLT_MAX ? copysignf(FLT_MAX, v) : v; }
template <typename T> __device__ __forceinline__ uint32_t pack2_saturated(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2_saturated<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2_saturated<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float load_scale(const void *scales, int64_t at, int e8m0) {
    if (!e8m0) return static_cast<const float *>(scales)[at];
    const uint32_t e = static_cast<const uint8_t *>(scales)[at];
    // 2^(e - 127); code 0 is the subnormal 2^-127, 255 is NaN
    return __uint_as_float(e == 0 ? 0x00400000u : e == 255 ? 0x7FC00000u : e << 23);
}

// N consecutive items at p, N * sizeof(T) <= 32 bytes and p aligned to it.
template <typename T, int N>
__device__ __forceinline__ void store_items(T *p, const float (&v)[N]) {
    if constexpr (N == 1) {
        if constexpr (sizeof(T) == 4) *p = saturated(v[0]);
        else *reinterpret_cast<uint16_t *>(p) = static_cast<uint16_t>(pack2_saturated<T>(v[0], 0.0f));
    } else {
        constexpr int W = N * sizeof(T) / 4;
        uint32_t w[W];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = __float_as_uint(saturated(v[j]));
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] = pack2_saturated<T>(v[2 * j], v[2 * j + 1]);
        }
        if constexpr (W == 8) {                    // sm_100's 256-bit store
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        } else {
            Chunk<uint32_t, W> c;
#pragma unroll
            for (int j = 0; j < W; ++j) c.word[j] = w[j];
            *reinterpret_cast<typename Chunk<uint32_t, W>::Word *>(p) = c.all;
        }
    }
}

template <typename T, int CV, int E5M2>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
    const ReadSide &s = p.side[blockIdx.y];
    __shared__ int64_t code_at[kTileRows], scale_at[kTileRows];
    __shared__ int state[kTileRows];               // 0: no row of a sequence, 1: zeros, 2: codes
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tile;
    if (threadIdx.x < p.tile) {
        const int64_t row = first + threadIdx.x;
        int now = 0;
        if (row < p.rows) {
            const int64_t b = paging::sequence_of_row(p.offsets, p.offset_bytes, p.seqs, row);
            if (b >= 0) {
                const paging::Place at = paging::place_in_sequence(
                    row - paging::load_index(p.offsets, p.offset_bytes, b), p.table, p.table_stride, p.table_width,
                    p.table_bytes, b, p.pages, p.page_size);
                now = at.ok ? 2 : 1;
                code_at[threadIdx.x] = at.page * s.code_page + at.slot * s.code_slot;
                scale_at[threadIdx.x] = at.page * s.scale_page + at.slot * s.scale_slot;
            }
        }
        state[threadIdx.x] = now;
    }
    __syncthreads();
    const int chunks = s.dim / CV, units = s.heads * chunks;          // chunks of a row's heads
    const int down = units < kThreads ? kThreads / units : 1;         // rows the block's threads cover at once
    const int across = units < kThreads ? units : kThreads;
    const int t0 = threadIdx.x / across;
    if (t0 >= down) return;
    for (int u = threadIdx.x - t0 * across; u < units; u += across) {
        const int head = u / chunks, d = (u - head * chunks) * CV;
        const uint8_t *codes = s.codes + head * s.code_head + d;
        const int64_t scales = head * s.scale_head + d / s.group;
        T *out = static_cast<T *>(s.out) + first * s.out_token + head * s.out_head + d;
        for (int t = t0; t < p.tile; t += kReadRows * down) {
            Chunk<uint8_t, CV> c[kReadRows];
            float scale[kReadRows];
            int now[kReadRows];
#pragma unroll
            for (int i = 0; i < kReadRows; ++i) {
                const int at = t + i * down;
                c[i] = Chunk<uint8_t, CV>{};
                scale[i] = 0.0f;
                now[i] = at < p.tile ? state[at] : 0;
                if (now[i] == 2) {
                    c[i] = load_chunk<uint8_t, CV>(codes + code_at[at]);
                    scale[i] = load_scale(s.scales, scales + scale_at[at], p.e8m0);
                }
            }
#pragma unroll
            for (int i = 0; i < kReadRows; ++i) {
                if (now[i] == 0) continue;
                float v[CV];
                if constexpr (CV == 1) {
                    v[0] = decode2<E5M2>(c[i].all).x * scale[i];
                } else {
#pragma unroll
                    for (int j = 0; j < CV / 4; ++j) {
                        const float2 f = decode2<E5M2>(static_cast<uint16_t>(c[i].word[j]));
                        const float2 h = decode2<E5M2>(static_cast<uint16_t>(c[i].word[j] >> 16));
                        const float2 by = make_float2(scale[i], scale[i]);
                        const float2 x = mul2(f, by), y = mul2(h, by);
                        v[4 * j] = x.x;
                        v[4 * j + 1] = x.y;
                        v[4 * j + 2] = y.x;
                        v[4 * j + 3] = y.y;
                    }
                }
                store_items<T, CV>(out + (t + i * down) * s.out_token, v);
            }
        }
    }
}

template <typename T, int CV>
void launch_read(const ReadParams &p, dim3 grid, cudaStream_t stream) {
    if (p.e5m2) cache_read_kernel<T, CV, 1><<<grid, kThreads, 0, stream>>>(p);
    else cache_read_kernel<T, CV, 0><<<grid, kThreads, 0, stream>>>(p);
}

// Widest chunk that a side's sizes, strides and addresses allow: 32 bytes of output at most.
int widest_read(const ReadSide &s, int itemsize) {
    for (int cv : {16, 8, 4}) {
        if (cv * itemsize > 32 || s.dim % cv || s.group % cv) continue;
        if ((reinterpret_cast<uintptr_t>(s.codes) | s.code_page | s.code_slot | s.code_head) % cv) continue;
        if (reinterpret_cast<uintptr_t>(s.out) % (cv * itemsize) || (s.out_token | s.out_head) % cv) continue;
        return cv;
    }
    return 1;
}

template <typename T>
void pick_read(const ReadParams &p, int cv, dim3 grid, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2)
        if (cv == 16) return launch_read<T, 16>(p, grid, stream);
    if (cv == 8) return launch_read<T, 8>(p, grid, stream);
    if (cv == 4) return launch_read<T, 4>(p, grid, stream);
    launch_read<T, 1>(p, grid, stream);
}

// Rows a block owns: smaller tiles where whole ones would leave SMs without a block (400
// rows of 8 heads of 128 items: 41 us with tiles of 32, 10.4 us so), or where a row is long
// work (16384 rows of 32 heads of 128 items: 81 us with tiles of 32, 70 us so; 6000 rows of 8
// heads of 33 items beside 128: 24.7 and 18.6).
int tile_rows(int64_t rows, int64_t chunks) {
    int tile = kTileRows;
    while (tile > 4 && (rows / tile < b2k::sm_count() || tile * chunks > 2048)) tile /= 2;
    return tile;
}

int check_sides_apart(const Params &p, const char *name) {
    if (int rc = check_apart(p.role[1].codes, p.role[2].codes, name, "the codes of keys and values")) return rc;
    return check_apart(p.role[1].scales, p.role[2].scales, name, "the scales of keys and values");
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
    if (int rc = check_sides_apart(p, name)) return rc;
    p.tokens = tokens;
    p.slots = slots_dev;
    p.slot_bytes = slot_bytes;
    return launch_forward<kWrite>(p, format, nullptr, b2k::as_stream(stream), name);
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
    if (cache->pages > 0)
        if (int rc = check_sides_apart(p, name)) return rc;
    p.tokens = r->tokens;
    p.slots = slots_dev;
    p.slot_bytes = slot_bytes;
    set_rotation(p, *r);
    return launch_forward<kBoth>(p, r->format, r, b2k::as_stream(stream), name);
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
    if (int rc = check_apart(p.side[0].out, p.side[1].out, name, "k_out and v_out")) return rc;
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
    const cudaStream_t st = b2k::as_stream(stream);
    int sides = 0, cv[2] = {};
    double items = 0;
    for (ReadSide &side : p.side) {                     // the sides that are there come first
        if (side.heads == 0) continue;
        items += static_cast<double>(rows) * side.heads * side.dim;
        cv[sides] = widest_read(side, item_bytes(format));
        p.side[sides++] = side;
    }
    // sides of different chunks: as in launch_forward
    const bool split = sides == 2 && cv[0] != cv[1] && items >= kItemsToSplit;
    if (sides == 2 && !split) cv[0] = cv[0] < cv[1] ? cv[0] : cv[1];
    // a thread's chunk number stays an int one step past the last chunk of a row
    for (int i = 0; i < sides; ++i)
        if (static_cast<int64_t>(p.side[i].heads) * p.side[i].dim / cv[split ? i : 0] > INT_MAX - kThreads)
            return b2k::fail(B2K_ERR_TOO_LARGE, "%s: a row has more than 2^31 - %d chunks", name, kThreads + 1);
    for (int i = 0; i < (split ? 2 : 1); ++i) {
        if (i) p.side[0] = p.side[1];
        const int here = split ? 1 : sides;
        int64_t chunks = 0;                                // of a row
        for (int k = 0; k < here; ++k)
            chunks = std::max<int64_t>(chunks, static_cast<int64_t>(p.side[k].heads) * p.side[k].dim / cv[i]);
        p.tile = tile_rows(rows, chunks);
        const int64_t blocks = (rows + p.tile - 1) / p.tile;
        if (blocks > INT_MAX) return b2k::fail(B2K_ERR_TOO_LARGE, "%s: too many rows for one launch", name);
        const dim3 grid(static_cast<unsigned>(blocks), here);
        if (format == B2K_FMT_F32) pick_read<float>(p, cv[i], grid, st);
        else if (format == B2K_FMT_F16) pick_read<__half>(p, cv[i], grid, st);
        else pick_read<__nv_bfloat16>(p, cv[i], grid, st);
        B2K_RETURN_IF_LAUNCH_FAILED(name);
        b2k::note_launch();
    }
    return B2K_OK;
}

}  // extern "C"
