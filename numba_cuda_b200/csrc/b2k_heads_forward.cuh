// The forward kernel of the head-wise family: norm, rotation and store or quantisation
// of rows, in one pass over the data.  MODE selects what a role may do, so that the
// plain cache write carries no rotation code and the plain rotation no quantisation.
#pragma once

#include "b2k_heads.cuh"

namespace headwise {

enum Mode { kRotate = 1, kWrite = 2, kBoth = 3 };

// Quantise one row held in registers into its cache slot.
template <int VEC, int ITER>
__device__ __forceinline__ void quantise_row(const Params &p, const Role &r, const Lanes &g,
                                             const paging::Place &at, int head, const float (&a)[ITER][VEC],
                                             const float (&b)[ITER][VEC], unsigned *group_max) {
    uint8_t *codes = r.codes + at.page * r.code_page + at.slot * r.code_slot + head * r.code_head;
    const int64_t scale_at = at.page * r.scale_page + at.slot * r.scale_slot + head * r.scale_head;
    const bool whole = r.group == r.dim;
    float row_scale = 1.0f, row_by = 1.0f;
    uint8_t code = 0;
    if (whole) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) m = fmaxf(m, fmaxf(largest_finite<VEC>(a[i]), largest_finite<VEC>(b[i])));
        row_scale = scale_for(g.max(m), p.e5m2, p.e8m0, code);
        row_by = __frcp_rn(row_scale);
        if (g.lane == 0) {
            if (p.e8m0) static_cast<uint8_t *>(r.scales)[scale_at] = code;
            else static_cast<float *>(r.scales)[scale_at] = row_scale;
        }
    } else {
        // the magnitudes' bit patterns are ordered like the magnitudes
        __syncwarp(g.mask);
        for (int k = g.lane; k < r.dim / r.group; k += g.n) group_max[k] = 0u;
        __syncwarp(g.mask);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            int oa, ob;
            unit_at<VEC>(r, g.lane + i * g.n, oa, ob);
            if (oa < r.dim) atomicMax(&group_max[oa / r.group], __float_as_uint(largest_finite<VEC>(a[i])));
            if (ob < r.dim) atomicMax(&group_max[ob / r.group], __float_as_uint(largest_finite<VEC>(b[i])));
        }
        __syncwarp(g.mask);
        for (int k = g.lane; k < r.dim / r.group; k += g.n) {
            const float s = scale_for(__uint_as_float(group_max[k]), p.e5m2, p.e8m0, code);
            if (p.e8m0) static_cast<uint8_t *>(r.scales)[scale_at + k] = code;
            else static_cast<float *>(r.scales)[scale_at + k] = s;
        }
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        int oa, ob;
        unit_at<VEC>(r, g.lane + i * g.n, oa, ob);
        float by_a = row_by, by_b = row_by;
        if (!whole) {
            if (oa < r.dim)
                by_a = __frcp_rn(scale_for(__uint_as_float(group_max[oa / r.group]), p.e5m2, p.e8m0, code));
            if (ob < r.dim)
                by_b = __frcp_rn(scale_for(__uint_as_float(group_max[ob / r.group]), p.e5m2, p.e8m0, code));
        }
        if (oa < r.dim) store_codes<VEC>(codes + oa, a[i], by_a, p.e5m2);
        if (ob < r.dim) store_codes<VEC>(codes + ob, b[i], by_b, p.e5m2);
    }
}

template <typename T, int VEC, int ITER, int MODE>
__global__ void __launch_bounds__(kThreads) heads_forward_kernel(const __grid_constant__ Params p) {
    // groups of a scale are at least 16 items, so a lane's share of a row has at most this many
    constexpr int kGroupsPerLane = (2 * VEC * ITER + 15) / 16;
    __shared__ unsigned group_max[MODE == kRotate ? 1 : kThreads * kGroupsPerLane];
    const Lanes g(p.lanes);
    const uint32_t in_block = static_cast<uint32_t>(kThreads) / static_cast<uint32_t>(g.n);
    const uint64_t wide = static_cast<uint64_t>(blockIdx.x) * in_block + threadIdx.x / static_cast<uint32_t>(g.n);
    if (wide >= p.items) return;                      // whole groups
    const uint32_t item = static_cast<uint32_t>(wide);
    const int64_t token = item / static_cast<uint32_t>(p.items_per_token);
    int part = static_cast<int>(item % static_cast<uint32_t>(p.items_per_token));
    int which = 0;
    while (part >= p.role[which].items) part -= p.role[which++].items;
    const Role &r = p.role[which];

    int64_t position = 0;
    if ((MODE & kRotate) && p.positions != nullptr) {
        position = paging::load_index(p.positions, p.position_bytes, token);
        if (position < 0 || position >= p.table_rows) return;
    }
    const bool quantised = MODE == kWrite || (MODE == kBoth && r.out == nullptr);
    paging::Place at{0, 0, false};
    if (quantised) {
        at = paging::place_of_slot(paging::load_index(p.slots, p.slot_bytes, token), p.pages, p.page_size);
        if (!at.ok) return;
    }
    const bool normed = (MODE & kRotate) && p.norm && which < 2;

    float c[ITER][VEC] = {}, s[ITER][VEC] = {}, wa[ITER][VEC] = {}, wb[ITER][VEC] = {};
    if constexpr ((MODE & kRotate) != 0) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int u = g.lane + i * g.n;
            if (u < r.angle_units) {
                load_floats<VEC>(p.cos_table + position * p.cos_stride + u * VEC, c[i]);
                load_floats<VEC>(p.sin_table + position * p.sin_stride + u * VEC, s[i]);
            }
            if (normed) {
                int oa, ob;
                unit_at<VEC>(r, u, oa, ob);
                if (oa < r.dim) load_weight<VEC>(r.weight, p.weight_format, oa, wa[i]);
                if (ob < r.dim) load_weight<VEC>(r.weight, p.weight_format, ob, wb[i]);
            }
        }
    }

    const int last = min(r.heads, (part + 1) * p.heads_per_item);
    for (int head = part * p.heads_per_item; head < last; ++head) {
        const T *in = static_cast<const T *>(r.in) + token * r.in_token + head * r.in_head;
        float a[ITER][VEC], b[ITER][VEC];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            int oa, ob;
            unit_at<VEC>(r, g.lane + i * g.n, oa, ob);
            Chunk<T, VEC> ca{}, cb{};
            if (oa < r.dim) ca = load_chunk<T, VEC>(in + oa);
            if (ob < r.dim) cb = load_chunk<T, VEC>(in + ob);
            widen(ca, a[i]);
            widen(cb, b[i]);
        }
        if constexpr ((MODE & kRotate) != 0) {
            if (normed) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < ITER; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ss += a[i][j] * a[i][j] + b[i][j] * b[i][j];
                const float by = rsqrtf(g.sum(ss) * r.inv_dim + p.eps);
#pragma unroll
                for (int i = 0; i < ITER; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        a[i][j] *= by * wa[i][j];
                        b[i][j] *= by * wb[i][j];
                    }
            }
#pragma unroll
            for (int i = 0; i < ITER; ++i)
                if (g.lane + i * g.n < r.angle_units) rotate<VEC>(a[i], b[i], c[i], s[i], p.interleaved);
        }
        if (!quantised) {
            T *out = static_cast<T *>(r.out) + token * r.out_token + head * r.out_head;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                int oa, ob;
                unit_at<VEC>(r, g.lane + i * g.n, oa, ob);
                if (oa < r.dim) store_chunk<T, VEC>(out + oa, a[i]);
                if (ob < r.dim) store_chunk<T, VEC>(out + ob, b[i]);
            }
        } else if constexpr (MODE != kRotate) {
            quantise_row<VEC, ITER>(p, r, g, at, head, a, b,
                                    group_max + (threadIdx.x & ~(g.n - 1)) * kGroupsPerLane);
        }
    }
}

// ---- launch --------------------------------------------------------------------------
template <typename T, int MODE>
void pick_forward(const Params &p, const Plan &plan, unsigned blocks, cudaStream_t stream) {
#define B2K_HEADS_CASE(V, I)                                                                 \
    if constexpr (V * sizeof(T) <= 16) if (plan.vec == V && plan.iter == I) { \
        heads_forward_kernel<T, V, I, MODE><<<blocks, kThreads, 0, stream>>>(p);             \
        return;                                                                              \
    }
    B2K_HEADS_SHAPES(B2K_HEADS_CASE)
#undef B2K_HEADS_CASE
}

// Launches over all items; the roles, tokens and tables of `p` are set.
template <int MODE>
int launch_forward(Params &p, int64_t format, const Plan &plan, cudaStream_t stream, const char *name) {
    if (int rc = count_items(p, name)) return rc;
    const int64_t in_block = kThreads / p.lanes;
    const int64_t blocks = (static_cast<int64_t>(p.items) + in_block - 1) / in_block;
    if (blocks == 0) return B2K_OK;
    if (blocks > INT_MAX) return b2k::fail(B2K_ERR_TOO_LARGE, "%s: too many rows for one launch", name);
    if (format == B2K_FMT_F32) pick_forward<float, MODE>(p, plan, static_cast<unsigned>(blocks), stream);
    else if (format == B2K_FMT_F16) pick_forward<__half, MODE>(p, plan, static_cast<unsigned>(blocks), stream);
    else pick_forward<__nv_bfloat16, MODE>(p, plan, static_cast<unsigned>(blocks), stream);
    B2K_RETURN_IF_LAUNCH_FAILED(name);
    b2k::note_launch();
    return B2K_OK;
}

}  // namespace headwise
