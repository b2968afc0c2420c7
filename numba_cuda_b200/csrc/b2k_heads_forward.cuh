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
        for (int i = 0; i < ITER; ++i) m = largest<VEC>(b[i], largest<VEC>(a[i], m));
        m = g.max(m, r.scale_lanes);
        if (__any_sync(g.mask, m > FLT_MAX)) {       // rare: again without the infinities
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < ITER; ++i) m = largest_finite<VEC>(b[i], largest_finite<VEC>(a[i], m));
            m = g.max(m, r.scale_lanes);
        }
        const Scale s(m, p.e5m2, p.e8m0);
        if ((g.lane & (r.scale_lanes - 1)) == 0 && oa[0] < r.dim) s.store(r.scales, scale_at + r.groups_of.quotient(oa[0]), p.e8m0);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < r.dim) store_codes<VEC>(codes + oa[i], a[i], s.inverse, p.e5m2);
            if (ob[i] < r.dim) store_codes<VEC>(codes + ob[i], b[i], s.inverse, p.e5m2);
        }
    } else if (ITER == 1 && r.scale_lanes) {
        float ma = g.max(largest<VEC>(a[0], 0.0f), r.scale_lanes), mb = g.max(largest<VEC>(b[0], 0.0f), r.scale_lanes);
        if (__any_sync(g.mask, fmaxf(ma, mb) > FLT_MAX)) {
            ma = g.max(largest_finite<VEC>(a[0], 0.0f), r.scale_lanes);
            mb = g.max(largest_finite<VEC>(b[0], 0.0f), r.scale_lanes);
        }
        const Scale sa(ma, p.e5m2, p.e8m0), sb(mb, p.e5m2, p.e8m0);
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
            if (oa[i] < r.dim) atomicMax(&group_max[r.groups_of.quotient(oa[i])], __float_as_uint(largest_finite<VEC>(a[i], 0.0f)));
            if (ob[i] < r.dim) atomicMax(&group_max[r.groups_of.quotient(ob[i])], __float_as_uint(largest_finite<VEC>(b[i], 0.0f)));
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

// A group's chunks of kRows rows of one token, as loaded.
template <typename T, int VEC, int ITER, int ROWS>
struct Batch {
    Chunk<T, VEC> a[ROWS][ITER], b[ROWS][ITER];
    __device__ __forceinline__ void load(const T *in, int64_t step, int rows, const int (&oa)[ITER], const int (&ob)[ITER],
                                         int dim) {
#pragma unroll
        for (int h = 0; h < ROWS; ++h)
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                a[h][i] = b[h][i] = Chunk<T, VEC>{};
                if (h < rows && oa[i] < dim) a[h][i] = load_chunk<T, VEC>(in + h * step + oa[i]);
                if (h < rows && ob[i] < dim) b[h][i] = load_chunk<T, VEC>(in + h * step + ob[i]);
            }
    }
};

// What the forward kernel multiplies a row's items by: k0 .. k3 of turn() for rotated
// units; k0 and k2 are the weights of the two chunks for the others.
template <int VEC, int ITER>
struct Factors {
    float k0[ITER][VEC], k1[ITER][VEC], k2[ITER][VEC], k3[ITER][VEC];
};

template <typename T, int VEC, int ITER, int MODE>
__global__ void __launch_bounds__(kThreads) heads_forward_kernel(const __grid_constant__ Params p) {
    // groups of a scale are at least 16 items, so a lane's share of a row has at most this many
    constexpr int kGroupsPerLane = (2 * VEC * ITER + 15) / 16;
    constexpr int kRows = rows_in_flight(ITER);
    __shared__ unsigned group_max[MODE == kRotate ? 1 : kThreads * kGroupsPerLane];
    // A block works for one role, so the role's members are uniform over the block.
    const uint32_t upto0 = p.role[0].blocks, upto1 = upto0 + p.role[1].blocks;
    const int which = (blockIdx.x >= upto0) + (blockIdx.x >= upto1);
    const uint32_t block = blockIdx.x - (which == 0 ? 0 : which == 1 ? upto0 : upto1);
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
    const T *in = static_cast<const T *>(r.in) + token * r.in_token + first * r.in_head;
    Batch<T, VEC, ITER, kRows> now;
    now.load(in, r.in_head, rows, oa, ob, r.dim);

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

    Factors<VEC, ITER> k;
    if constexpr ((MODE & kRotate) != 0) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int u = g.lane + i * g.n;
            float wa[VEC], wb[VEC], c[VEC], s[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) wa[j] = wb[j] = 1.0f;
            if (normed && oa[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, oa[i], wa);
            if (normed && ob[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, ob[i], wb);
            if (u < r.angle_units) {
                load_floats<VEC>(p.cos_table + position * p.cos_stride + u * VEC, c);
                load_floats<VEC>(p.sin_table + position * p.sin_stride + u * VEC, s);
                float wx[VEC], wy[VEC];
                if (p.interleaved) {
                    pair<VEC>(wa, wb, wx, wy);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        wx[j] = wa[j];
                        wy[j] = wb[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    k.k0[i][j] = wx[j] * c[j];
                    k.k1[i][j] = wy[j] * s[j];
                    k.k2[i][j] = wy[j] * c[j];
                    k.k3[i][j] = wx[j] * s[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    k.k0[i][j] = wa[j];
                    k.k2[i][j] = wb[j];
                    k.k1[i][j] = k.k3[i][j] = 0.0f;
                }
            }
        }
    }

#pragma unroll 1
    for (int done = 0; done < rows; done += kRows) {
        // the next rows are on their way while these are worked on
        Batch<T, VEC, ITER, kRows> next;
        in += kRows * r.in_head;
        next.load(in, r.in_head, rows - done - kRows, oa, ob, r.dim);
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            if (done + h >= rows) break;
            float a[ITER][VEC], b[ITER][VEC];
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                widen(now.a[h][i], a[i]);
                widen(now.b[h][i], b[i]);
            }
            if constexpr ((MODE & kRotate) != 0) {
                float by = 1.0f;
                if (normed) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < ITER; ++i) ss = squares<VEC>(a[i], b[i], ss);
                    by = rsqrtf(g.sum(ss) * r.inv_dim + p.eps);
                }
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    if (g.lane + i * g.n < r.angle_units) {
                        if (p.interleaved) {
                            float x[VEC], y[VEC];
                            pair<VEC>(a[i], b[i], x, y);
                            turn<VEC>(x, y, k.k0[i], k.k1[i], k.k2[i], k.k3[i], by);
                            unpair<VEC>(x, y, a[i], b[i]);
                        } else {
                            turn<VEC>(a[i], b[i], k.k0[i], k.k1[i], k.k2[i], k.k3[i], by);
                        }
                    } else if (normed) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            a[i][j] *= by * k.k0[i][j];
                            b[i][j] *= by * k.k2[i][j];
                        }
                    }
                }
            }
            const int head = first + done + h;
            if (!quantised) {
                T *out = static_cast<T *>(r.out) + token * r.out_token + head * r.out_head;
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    if (oa[i] < r.dim) store_chunk<T, VEC>(out + oa[i], a[i]);
                    if (ob[i] < r.dim) store_chunk<T, VEC>(out + ob[i], b[i]);
                }
            } else if constexpr (MODE != kRotate) {
                quantise_row<VEC, ITER>(p, r, g, at, head, a, b, group_max + (threadIdx.x & ~(g.n - 1)) * kGroupsPerLane);
            }
        }
        now = next;
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
    if (int rc = count_items(p, kHeadsPerItem, kThreads, name)) return rc;
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
