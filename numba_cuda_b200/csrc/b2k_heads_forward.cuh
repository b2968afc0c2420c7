// The forward kernel of the head-wise family: norm, rotation and store or quantisation
// of rows, in one pass over the data.  MODE selects what a role may do, so that the
// plain cache write carries no rotation code and the plain rotation no quantisation.
#pragma once

#include "b2k_heads.cuh"

namespace headwise {

enum Mode { kRotate = 1, kWrite = 2, kBoth = 3 };

// Quantise one row held in registers into its cache slot.
template <int VEC, int ITER>
__device__ __forceinline__ void quantise_row(const Params &p, const Role &r, const Lanes &g, const paging::Place &at,
                                             int head, const float (&a)[ITER][VEC], const float (&b)[ITER][VEC],
                                             unsigned *group_max) {
    uint8_t *codes = r.codes + at.page * r.code_page + at.slot * r.code_slot + head * r.code_head;
    const int64_t scale_at = at.page * r.scale_page + at.slot * r.scale_slot + head * r.scale_head;
    int oa[ITER], ob[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) unit_at<VEC>(r, g.lane + i * g.n, oa[i], ob[i]);
    if (r.scale_lanes && r.scale_joint) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) m = fmaxf(m, fmaxf(largest_finite<VEC>(a[i]), largest_finite<VEC>(b[i])));
        const Scale s(g.max(m, r.scale_lanes), p.e5m2, p.e8m0);
        if ((g.lane & (r.scale_lanes - 1)) == 0 && oa[0] < r.dim) s.store(r.scales, scale_at + r.groups_of.quotient(oa[0]), p.e8m0);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < r.dim) store_codes<VEC>(codes + oa[i], a[i], s.inverse, p.e5m2);
            if (ob[i] < r.dim) store_codes<VEC>(codes + ob[i], b[i], s.inverse, p.e5m2);
        }
    } else if (ITER == 1 && r.scale_lanes) {
        const Scale sa(g.max(largest_finite<VEC>(a[0]), r.scale_lanes), p.e5m2, p.e8m0);
        const Scale sb(g.max(largest_finite<VEC>(b[0]), r.scale_lanes), p.e5m2, p.e8m0);
        if ((g.lane & (r.scale_lanes - 1)) == 0 && oa[0] < r.dim) {
            sa.store(r.scales, scale_at + r.groups_of.quotient(oa[0]), p.e8m0);
            sb.store(r.scales, scale_at + r.groups_of.quotient(ob[0]), p.e8m0);
        }
        if (oa[0] < r.dim) {
            store_codes<VEC>(codes + oa[0], a[0], sa.inverse, p.e5m2);
            store_codes<VEC>(codes + ob[0], b[0], sb.inverse, p.e5m2);
        }
    } else {
        // any other layout of groups: the magnitudes' bit patterns are ordered like the
        // magnitudes, so an integer maximum in shared memory finds them
        const int groups = r.groups_of.quotient(r.dim);
        __syncwarp(g.mask);
        for (int k = g.lane; k < groups; k += g.n) group_max[k] = 0u;
        __syncwarp(g.mask);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < r.dim) atomicMax(&group_max[r.groups_of.quotient(oa[i])], __float_as_uint(largest_finite<VEC>(a[i])));
            if (ob[i] < r.dim) atomicMax(&group_max[r.groups_of.quotient(ob[i])], __float_as_uint(largest_finite<VEC>(b[i])));
        }
        __syncwarp(g.mask);
        for (int k = g.lane; k < groups; k += g.n)
            Scale(__uint_as_float(group_max[k]), p.e5m2, p.e8m0).store(r.scales, scale_at + k, p.e8m0);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < r.dim)
                store_codes<VEC>(codes + oa[i], a[i],
                                 Scale(__uint_as_float(group_max[r.groups_of.quotient(oa[i])]), p.e5m2, p.e8m0).inverse, p.e5m2);
            if (ob[i] < r.dim)
                store_codes<VEC>(codes + ob[i], b[i],
                                 Scale(__uint_as_float(group_max[r.groups_of.quotient(ob[i])]), p.e5m2, p.e8m0).inverse, p.e5m2);
        }
    }
}

template <typename T, int VEC, int ITER, int MODE>
__global__ void __launch_bounds__(kThreads) heads_forward_kernel(const __grid_constant__ Params p) {
    // groups of a scale are at least 16 items, so a lane's share of a row has at most this many
    constexpr int kGroupsPerLane = (2 * VEC * ITER + 15) / 16;
    constexpr int kRows = rows_in_flight(ITER);
    __shared__ unsigned group_max[MODE == kRotate ? 1 : kThreads * kGroupsPerLane];
    // A block works for one role, so the role's members are uniform over the block.
    uint32_t block = blockIdx.x;
    int which = 0;
    while (block >= p.role[which].blocks) block -= p.role[which++].blocks;
    const Role &r = p.role[which];
    const Lanes g(p.lanes);
    const uint32_t item = block * (static_cast<uint32_t>(kThreads) >> p.lane_bits) + (threadIdx.x >> p.lane_bits);
    if (item >= r.all_items) return;                  // whole groups
    const uint32_t at_token = r.items.quotient(item);
    const int64_t token = at_token;
    const int part = static_cast<int>(item - at_token * r.items.d);
    const int first = part * p.heads_per_item;
    const int rows = min(r.heads - first, p.heads_per_item);
    int oa[ITER], ob[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) unit_at<VEC>(r, g.lane + i * g.n, oa[i], ob[i]);

    // The rows' loads go first: they do not wait for the token's position and slot.
    Chunk<T, VEC> ca[kRows][ITER], cb[kRows][ITER];
    const T *in = static_cast<const T *>(r.in) + token * r.in_token + first * r.in_head;
#pragma unroll
    for (int h = 0; h < kRows; ++h)
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            ca[h][i] = cb[h][i] = Chunk<T, VEC>{};
            if (h < rows && oa[i] < r.dim) ca[h][i] = load_chunk<T, VEC>(in + h * r.in_head + oa[i]);
            if (h < rows && ob[i] < r.dim) cb[h][i] = load_chunk<T, VEC>(in + h * r.in_head + ob[i]);
        }

    const bool quantised = MODE == kWrite || (MODE == kBoth && r.out == nullptr);
    int64_t position = 0, slot = 0;
    if (quantised) slot = paging::load_index(p.slots, p.slot_bytes, token);
    if ((MODE & kRotate) && p.positions != nullptr) {
        position = paging::load_index(p.positions, p.position_bytes, token);
        if (position < 0 || position >= p.table_rows) return;
    }
    paging::Place at{0, 0, false};
    if (quantised) {
        at = paging::place_of_slot(slot, p.pages, p.page_size);
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
                if (oa[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, oa[i], wa[i]);
                if (ob[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, ob[i], wb[i]);
            }
        }
    }

#pragma unroll
    for (int h = 0; h < kRows; ++h) {
        if (h >= rows) break;
        float a[ITER][VEC], b[ITER][VEC];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            widen(ca[h][i], a[i]);
            widen(cb[h][i], b[i]);
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
            T *out = static_cast<T *>(r.out) + token * r.out_token + (first + h) * r.out_head;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                if (oa[i] < r.dim) store_chunk<T, VEC>(out + oa[i], a[i]);
                if (ob[i] < r.dim) store_chunk<T, VEC>(out + ob[i], b[i]);
            }
        } else if constexpr (MODE != kRotate) {
            quantise_row<VEC, ITER>(p, r, g, at, first + h, a, b,
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
    if (int rc = count_items(p, rows_in_flight(plan.iter), kThreads, name)) return rc;
    const unsigned blocks = p.role[0].blocks + p.role[1].blocks + p.role[2].blocks;
    if (blocks == 0) return B2K_OK;
    if (format == B2K_FMT_F32) pick_forward<float, MODE>(p, plan, blocks, stream);
    else if (format == B2K_FMT_F16) pick_forward<__half, MODE>(p, plan, blocks, stream);
    else pick_forward<__nv_bfloat16, MODE>(p, plan, blocks, stream);
    B2K_RETURN_IF_LAUNCH_FAILED(name);
    b2k::note_launch();
    return B2K_OK;
}

}  // namespace headwise
