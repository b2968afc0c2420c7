// The forward kernel of the head-wise family: norm, rotation and store or quantisation
// of rows, in one pass over the data.  MODE selects what a role may do, so that the
// plain cache write carries no rotation code and the plain rotation no quantisation.
#pragma once

#include "b2k_heads.cuh"

namespace headwise {

enum Mode { kRotate = 1, kWrite = 2, kBoth = 3 };

// Quantise one row held in registers into its cache slot: `codes` and `scale_at` are the
// row's place, oa and ob where the lane's chunks start.
template <int VEC, int ITER>
__device__ __forceinline__ void quantise_row(const Params &p, const Role &r, const Lanes &g, uint8_t *codes,
                                             int64_t scale_at, const int (&oa)[ITER], const int (&ob)[ITER],
                                             const float (&a)[ITER][VEC], const float (&b)[ITER][VEC],
                                             unsigned *group_max, bool there) {
    const int dim = there ? r.dim : 0;         // a row that is not there stores nothing
    if (r.scale_lanes && r.scale_joint) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) m = largest<VEC>(b[i], largest<VEC>(a[i], m));
        m = g.max(m, r.scale_lanes);
        if (__any_sync(0xFFFFFFFFu, m > FLT_MAX)) {       // rare: again without the infinities
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < ITER; ++i) m = largest_finite<VEC>(b[i], largest_finite<VEC>(a[i], m));
            m = g.max(m, r.scale_lanes);
        }
        const Scale s(m, p.e5m2, p.e8m0);
        if ((g.lane & (r.scale_lanes - 1)) == 0 && oa[0] < dim) s.store(r.scales, scale_at + r.groups_of.quotient(oa[0]), p.e8m0);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < dim) store_codes<VEC>(codes + oa[i], a[i], s.inverse, p.e5m2);
            if (ob[i] < dim) store_codes<VEC>(codes + ob[i], b[i], s.inverse, p.e5m2);
        }
    } else if (ITER == 1 && r.scale_lanes) {
        float ma = g.max(largest<VEC>(a[0], 0.0f), r.scale_lanes), mb = g.max(largest<VEC>(b[0], 0.0f), r.scale_lanes);
        if (__any_sync(0xFFFFFFFFu, fmaxf(ma, mb) > FLT_MAX)) {
            ma = g.max(largest_finite<VEC>(a[0], 0.0f), r.scale_lanes);
            mb = g.max(largest_finite<VEC>(b[0], 0.0f), r.scale_lanes);
        }
        const Scale sa(ma, p.e5m2, p.e8m0), sb(mb, p.e5m2, p.e8m0);
        if ((g.lane & (r.scale_lanes - 1)) == 0 && oa[0] < dim) {
            sa.store(r.scales, scale_at + r.groups_of.quotient(oa[0]), p.e8m0);
            sb.store(r.scales, scale_at + r.groups_of.quotient(ob[0]), p.e8m0);
        }
        if (oa[0] < dim) {
            store_codes<VEC>(codes + oa[0], a[0], sa.inverse, p.e5m2);
            store_codes<VEC>(codes + ob[0], b[0], sb.inverse, p.e5m2);
        }
    } else {
        // any other layout of groups: the magnitudes' bit patterns are ordered like the
        // magnitudes, so an integer maximum in shared memory finds them
        const int groups = r.groups_of.quotient(r.dim);
        __syncwarp();
        for (int k = g.lane; k < groups; k += g.n) group_max[k] = 0u;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < dim) atomicMax(&group_max[r.groups_of.quotient(oa[i])], __float_as_uint(largest_finite<VEC>(a[i], 0.0f)));
            if (ob[i] < dim) atomicMax(&group_max[r.groups_of.quotient(ob[i])], __float_as_uint(largest_finite<VEC>(b[i], 0.0f)));
        }
        __syncwarp();
        for (int k = g.lane; k < groups && there; k += g.n)
            Scale(__uint_as_float(group_max[k]), p.e5m2, p.e8m0).store(r.scales, scale_at + k, p.e8m0);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if (oa[i] < dim)
                store_codes<VEC>(codes + oa[i], a[i],
                                 Scale(__uint_as_float(group_max[r.groups_of.quotient(oa[i])]), p.e5m2, p.e8m0).inverse, p.e5m2);
            if (ob[i] < dim)
                store_codes<VEC>(codes + ob[i], b[i],
                                 Scale(__uint_as_float(group_max[r.groups_of.quotient(ob[i])]), p.e5m2, p.e8m0).inverse, p.e5m2);
        }
    }
}

// What the forward kernel multiplies a row's pairs by: k0 .. k3 of turn().
template <int VEC, int ITER>
struct Factors {
    float k0[ITER][VEC], k1[ITER][VEC], k2[ITER][VEC], k3[ITER][VEC];
};

// One role's share of the launch.  WHICH is a constant so that every member of the role is
// an operand in constant memory: indexed by a variable, each use is a load of its own,
// and those were a quarter of all instructions.
template <typename T, int VEC, int ITER, int MODE, int WHICH, bool INTER>
__device__ __forceinline__ void forward_role(const Params &p, uint32_t block, unsigned *group_max) {
    // groups of a scale are at least 16 items, so a lane's share of a row has at most this many
    constexpr int kGroupsPerLane = (2 * VEC * ITER + 15) / 16;
    constexpr int kRows = rows_in_flight(ITER);
    constexpr bool rotates = (MODE & kRotate) != 0 && WHICH < 2;
    constexpr bool quantised = (MODE & kWrite) != 0 && WHICH > 0;
    const Role &r = p.role[WHICH];
    const Lanes g(p.lanes);
    const uint32_t item = block * (static_cast<uint32_t>(kThreads) >> p.lane_bits) + (threadIdx.x >> p.lane_bits);
    bool active = item < r.all_items;                  // the same for a whole group
    const uint32_t at_token = active ? r.items.quotient(item) : 0;
    const int64_t token = at_token;
    const int first = active ? static_cast<int>(item - at_token * r.items.d) * r.heads_per_item : 0;
    int rows = active ? min(r.heads - first, r.heads_per_item) : 0;
    int oa[ITER], ob[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) unit_at<VEC>(r, g.lane + i * g.n, oa[i], ob[i]);

    // The rows' loads go first: they do not wait for the token's position and slot.
    const T *in = static_cast<const T *>(r.in) + token * r.in_token + first * r.in_head;
    Batch<T, VEC, ITER, kRows> now;
    now.load(in, r.in_head, rows, oa, ob, r.dim);

    int64_t position = 0, slot = 0;
    if constexpr (quantised) slot = paging::load_index(p.slots, p.slot_bytes, token);
    if ((MODE & kRotate) && p.positions != nullptr) {
        position = paging::load_index(p.positions, p.position_bytes, token);
        active = active && position >= 0 && position < p.table_rows;
        if (!active) position = 0;
    }
    uint8_t *codes = nullptr;
    int64_t scale_at = 0;
    T *out = nullptr;
    if constexpr (quantised) {
        const paging::Place at = paging::place_of_slot(slot, p.pages, p.page_size);
        active = active && at.ok;
        codes = r.codes + at.page * r.code_page + at.slot * r.code_slot + first * r.code_head;
        scale_at = at.page * r.scale_page + at.slot * r.scale_slot + first * r.scale_head;
    } else {
        out = static_cast<T *>(r.out) + token * r.out_token + first * r.out_head;
    }
    const bool normed = rotates && p.norm;

    Factors<VEC, ITER> k;
    if constexpr (rotates) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int u = g.lane + i * g.n;
            const Turned t = turned_of<VEC, INTER>(r, u, oa[i], ob[i]);
            float wa[VEC], wb[VEC], wx[VEC], wy[VEC], c[VEC], s[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) wa[j] = wb[j] = 1.0f;
            if (normed && oa[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, oa[i], wa);
            if (normed && ob[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, ob[i], wb);
            in_pairs<VEC, INTER>(wa, wb, wx, wy);
            const Turned load{t.lo && active, t.hi && active};
            load_angles<VEC, INTER>(p.cos_table + position * p.cos_stride, u, oa[i], ob[i], load, c);
            load_angles<VEC, INTER>(p.sin_table + position * p.sin_stride, u, oa[i], ob[i], load, s);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const bool turned = j < VEC / 2 ? t.lo : t.hi;
                k.k0[i][j] = turned ? wx[j] * c[j] : wx[j];
                k.k1[i][j] = wy[j] * s[j];
                k.k2[i][j] = turned ? wy[j] * c[j] : wy[j];
                k.k3[i][j] = wx[j] * s[j];
            }
        }
    }

    if (!active) rows = 0;
    const int most = __reduce_max_sync(0xFFFFFFFFu, rows);
#pragma unroll 1
    for (int done = 0; done < most; done += kRows) {
        // the next rows are on their way while these are worked on
        Batch<T, VEC, ITER, kRows> next;
        in += kRows * r.in_head;
        next.load(in, r.in_head, rows - done - kRows, oa, ob, r.dim);
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            const bool there = done + h < rows;
            float a[ITER][VEC], b[ITER][VEC];
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                widen(now.a[h][i], a[i]);
                widen(now.b[h][i], b[i]);
            }
            if constexpr (rotates) {
                float by = 1.0f;
                if (normed) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < ITER; ++i) ss = squares<VEC>(a[i], b[i], ss);
                    by = rsqrtf(g.sum(ss) * r.inv_dim + p.eps);
                }
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    const Turned t = turned_of<VEC, INTER>(r, g.lane + i * g.n, oa[i], ob[i]);
                    float x[VEC], y[VEC];
                    in_pairs<VEC, INTER>(a[i], b[i], x, y);
                    if (VEC > 1) turn<0, VEC / 2, VEC>(x, y, k.k0[i], k.k1[i], k.k2[i], k.k3[i], by, t.lo);
                    turn<VEC / 2, VEC, VEC>(x, y, k.k0[i], k.k1[i], k.k2[i], k.k3[i], by, t.hi);
                    out_of_pairs<VEC, INTER>(x, y, a[i], b[i]);
                }
            }
            if constexpr (quantised) {
                quantise_row<VEC, ITER>(p, r, g, codes, scale_at, oa, ob, a, b,
                                        group_max + (threadIdx.x & ~(g.n - 1)) * kGroupsPerLane, there);
                codes += r.code_head;
                scale_at += r.scale_head;
            } else {
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    if (there && oa[i] < r.dim) store_chunk<T, VEC>(out + oa[i], a[i]);
                    if (there && ob[i] < r.dim) store_chunk<T, VEC>(out + ob[i], b[i]);
                }
                out += r.out_head;
            }
        }
        now = next;
    }
}

template <typename T, int VEC, int ITER, int MODE, bool INTER>
__device__ __forceinline__ void forward_roles(const Params &p, unsigned *group_max) {
    uint32_t block = blockIdx.x;
    if constexpr ((MODE & kRotate) != 0) {                 // a cache write has no queries
        if (block < p.role[0].blocks) return forward_role<T, VEC, ITER, MODE, 0, INTER>(p, block, group_max);
        block -= p.role[0].blocks;
    }
    if (MODE == kRotate || block < p.role[1].blocks) return forward_role<T, VEC, ITER, MODE, 1, INTER>(p, block, group_max);
    if constexpr (MODE != kRotate) forward_role<T, VEC, ITER, MODE, 2, INTER>(p, block - p.role[1].blocks, group_max);
}

// Five blocks an SM where a row takes one unit a lane (96 registers): left alone the compiler
// takes a few more and four fit (rotation of 16384 tokens x 40 heads of 128 bf16 items 66 us
// instead of 62 us).  The joined step of 16-bit items spills 56 bytes under this bound; four
// blocks were not measured for it.
template <typename T, int VEC, int ITER, int MODE>
__global__ void __launch_bounds__(kThreads, ITER == 1 ? 5 : 1) heads_forward_kernel(const __grid_constant__ Params p) {
    __shared__ unsigned group_max[MODE == kRotate ? 1 : kThreads * ((2 * VEC * ITER + 15) / 16)];
    if constexpr ((MODE & kRotate) != 0 && VEC > 1) {
        if (p.interleaved) return forward_roles<T, VEC, ITER, MODE, true>(p, group_max);
    }
    forward_roles<T, VEC, ITER, MODE, false>(p, group_max);
}

// ---- launch --------------------------------------------------------------------------
template <typename T, int MODE>
void pick_forward(const Params &p, const Plan &plan, unsigned blocks, cudaStream_t stream) {
#define B2K_HEADS_CASE(V, I)                                                                 \
    if constexpr (V * sizeof(T) <= 16)                                                       \
        if (plan.vec == V && plan.iter == I)                                                 \
            return heads_forward_kernel<T, V, I, MODE><<<blocks, kThreads, 0, stream>>>(p);
    B2K_HEADS_SHAPES(B2K_HEADS_CASE)
#undef B2K_HEADS_CASE
}

// 1024 tokens x 40 heads of 128 bf16 items: 6.8 us, with 256 8.0, with 1024 8.3, with 2048
// 12.4; 2048 tokens: 9.5, 11.3, 10.5, 12.8.  Not measured for other types and heads.
constexpr int kForwardBusy = 512;

// Roles whose sizes or strides allow different chunks get launches of their own when they
// hold at least this many items together.  Cache write, 8 heads of 128 bf16 items for keys
// and of 33 for values, in one launch and in two: 1.0 million items 8.3 and 10.4 us, 2.1
// million 12.4 and 11.4, 7.7 million 30.9 and 20.5.
constexpr int64_t kItemsToSplit = int64_t(1) << 20;

// Launches over all items; the roles, tokens and tables of `p` are set.
template <int MODE>
int launch_forward(const Params &all, int64_t format, const b2k_rotation *rot, cudaStream_t stream, const char *name) {
    int vec[3] = {}, least = 8, most = 0;
    double items = 0;
    for (int i = 0; i < 3; ++i) {
        const Role &r = all.role[i];
        if (r.heads == 0) continue;
        vec[i] = widest(all, i, format, rot);
        if (vec[i] < least) least = vec[i];
        if (vec[i] > most) most = vec[i];
        items += static_cast<double>(all.tokens) * r.heads * r.dim;
    }
    const bool split = least != most && items >= kItemsToSplit;
    for (int width : {8, 4, 2, 1}) {
        // the roles of this width, or all of them at the least
        if (split ? vec[0] != width && vec[1] != width && vec[2] != width : width != least || most == 0) continue;
        Params p = all;
        for (int i = 0; i < 3; ++i)
            if (split && vec[i] != width) p.role[i].heads = 0;
        const Plan plan = lay_out(p, width, rot);
        if (plan.iter == 0) return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: no kernel for this head size", name);
        if (int rc = count_items(p, kHeadsPerItem, kForwardBusy, name)) return rc;
        if (int rc = check_apart(all.role[0].out, all.role[1].out, name, "q_out and k_out")) return rc;
        const unsigned blocks = p.role[0].blocks + p.role[1].blocks + p.role[2].blocks;
        if (format == B2K_FMT_F32) pick_forward<float, MODE>(p, plan, blocks, stream);
        else if (format == B2K_FMT_F16) pick_forward<__half, MODE>(p, plan, blocks, stream);
        else pick_forward<__nv_bfloat16, MODE>(p, plan, blocks, stream);
        B2K_RETURN_IF_LAUNCH_FAILED(name);
        b2k::note_launch();
    }
    return B2K_OK;
}

}  // namespace headwise
