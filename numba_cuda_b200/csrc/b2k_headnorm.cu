// Norm and rotation of queries and keys, head by head, forward and backward, and the
// argument checks and layout choices shared with the cache kernels (b2k_kvcache.cu).
//
//   forward   y = R(x r w),  r = 1 / sqrt(mean(x^2) + eps),  R the rotation of the
//             position's angles
//   backward  g = R^T dy,  h = g w,  n = x r
//             dx = r (h - n mean(h n)),   dw = sum over tokens and heads of g n
//
// Both are one pass: a row is read once, stays in registers, and is written once, so
// HBM bounds them (2 and 3 items moved per item of the rows).  Sums are kept in float32
// and a value is rounded once, when it is stored.  Measured with bf16 items, 32 + 8 heads
// of 128: forward, 16384 tokens, 62 us = 5.6 TB/s (a copy of the same bytes 60 us);
// backward, 32768 tokens, 176 to 188 us on different GPUs = 5.4 to 5.8 TB/s with inputs that
// change from call to call (173 us on three sets of inputs in turn; a copy 164 us).  The
// reference's users would write this as a last-axis reduction of their own; its library reduce
// stops at one axis (numba/cuda/kernels/reduction.py:217-218).
#include <algorithm>

#include "b2k_heads_forward.cuh"

namespace headwise {

// ---- argument checks ---------------------------------------------------------------
int item_bytes(int64_t format) {
    if (format == B2K_FMT_F32) return 4;
    if (format == B2K_FMT_F16 || format == B2K_FMT_BF16) return 2;
    return 0;
}

// Whether an array of `n` axes (outer sizes and strides, innermost run of `run` items)
// has two items at one address; sizes <= 1 do not count.
static bool overlapping(int n, const int64_t *size, const int64_t *stride, int64_t run) {
    int order[4];
    int m = 0;
    for (int i = 0; i < n; ++i)
        if (size[i] > 1) order[m++] = i;
    for (int i = 1; i < m; ++i)
        for (int j = i; j > 0 && llabs(stride[order[j]]) < llabs(stride[order[j - 1]]); --j) {
            const int t = order[j];
            order[j] = order[j - 1];
            order[j - 1] = t;
        }
    int64_t span = run;
    for (int i = 0; i < m; ++i) {
        const int64_t step = llabs(stride[order[i]]);
        if (step < span) return true;
        span = step * (size[order[i]] - 1) + span;
    }
    return false;
}

int check_tokens(int64_t format, int64_t tokens, const char *name) {
    if (item_bytes(format) == 0) return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: items must be f32, f16 or bf16", name);
    if (tokens < 0) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: negative number of tokens", name);
    return B2K_OK;
}

int check_heads(const b2k_heads &h, const char *name, const char *what, int64_t tokens, int itemsize, bool written) {
    if (h.heads < 0 || h.heads > INT_MAX)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s has an invalid number of heads", name, what);
    if (h.heads == 0) return B2K_OK;
    if (h.dim < 1) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s has no items in a head", name, what);
    if (h.dim > B2K_MAX_HEAD_DIM)
        return b2k::fail(B2K_ERR_TOO_LARGE, "%s: %s has heads of more than %d items", name, what, B2K_MAX_HEAD_DIM);
    if (h.heads > INT_MAX / h.dim)
        return b2k::fail(B2K_ERR_TOO_LARGE, "%s: a token of %s has more than 2^31 - 1 items", name, what);
    if (tokens == 0) return B2K_OK;
    if (h.data_dev == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s is a null pointer", name, what);
    if (reinterpret_cast<uintptr_t>(h.data_dev) % itemsize)
        return b2k::fail(B2K_ERR_ALIGNMENT, "%s: %s is not aligned to its items", name, what);
    const int64_t size[2] = {tokens, h.heads}, stride[2] = {h.token_stride, h.head_stride};
    if (written && overlapping(2, size, stride, h.dim))
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: rows of %s overlap", name, what);
    return B2K_OK;
}

int check_apart(const void *a, const void *b, const char *name, const char *what) {
    if (a != nullptr && a == b) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s are the same memory", name, what);
    return B2K_OK;
}

int check_like(const b2k_heads &h, const b2k_heads &like, const char *name, const char *what) {
    if (h.heads != like.heads || (h.heads && h.dim != like.dim))
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s has another shape than its input", name, what);
    return B2K_OK;
}

int check_indices(const void *p, int64_t bytes, const char *name, const char *what) {
    if (bytes != 4 && bytes != 8)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s must be 4 or 8 byte integers", name, what);
    if (p == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: %s is a null pointer", name, what);
    if (reinterpret_cast<uintptr_t>(p) % bytes)
        return b2k::fail(B2K_ERR_ALIGNMENT, "%s: %s is not aligned to its items", name, what);
    return B2K_OK;
}

// Positions tell padding tokens even where nothing is rotated.
static bool has_positions(const b2k_rotation &r) { return r.rotary_dim > 0 || r.positions_dev != nullptr; }

int check_rotation(const b2k_rotation *r, const char *name) {
    if (r == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    if (int rc = check_tokens(r->format, r->tokens, name)) return rc;
    const int itemsize = item_bytes(r->format);
    if (int rc = check_heads(r->q, name, "q", r->tokens, itemsize, false)) return rc;
    if (int rc = check_heads(r->k, name, "k", r->tokens, itemsize, false)) return rc;
    if (r->norm != 0 && r->norm != 1) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: norm must be 0 or 1", name);
    if (r->norm) {
        if (!(r->eps >= 0.0)) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: eps must not be negative", name);
        const int wbytes = item_bytes(r->weight_format);
        if ((r->q_weight_dev || r->k_weight_dev) && wbytes == 0)
            return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: weights must be f32, f16 or bf16", name);
        for (const void *w : {r->q_weight_dev, r->k_weight_dev})
            if (w && reinterpret_cast<uintptr_t>(w) % wbytes)
                return b2k::fail(B2K_ERR_ALIGNMENT, "%s: a weight is not aligned to its items", name);
    }
    if (r->interleaved != 0 && r->interleaved != 1)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: interleaved must be 0 or 1", name);
    if (r->rotary_dim < 0 || r->rotary_dim % 2)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: rotary_dim must be even and not negative", name);
    if (r->rotary_dim > 0) {
        for (const b2k_heads *h : {&r->q, &r->k})
            if (h->heads && r->rotary_dim > h->dim)
                return b2k::fail(B2K_ERR_INVALID_ARG, "%s: rotary_dim is larger than a head", name);
        if (r->tokens > 0) {
            if (r->table_rows > 0 && (r->cos_dev == nullptr || r->sin_dev == nullptr))
                return b2k::fail(B2K_ERR_INVALID_ARG, "%s: cos or sin is a null pointer", name);
            for (const void *t : {r->cos_dev, r->sin_dev})
                if (reinterpret_cast<uintptr_t>(t) % 4)
                    return b2k::fail(B2K_ERR_ALIGNMENT, "%s: cos or sin is not aligned to its items", name);
        }
    }
    if (has_positions(*r)) {
        if (r->table_rows < 0) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: negative table_rows", name);
        if (r->tokens > 0)
            if (int rc = check_indices(r->positions_dev, r->position_bytes, name, "positions")) return rc;
    }
    return B2K_OK;
}

int check_cache(const b2k_cache *c, const char *name) {
    if (c == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null cache", name);
    if (c->code_format != B2K_FMT_E4M3 && c->code_format != B2K_FMT_E5M2)
        return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: codes must be e4m3 or e5m2", name);
    if (c->scale_format != B2K_FMT_F32 && c->scale_format != B2K_FMT_E8M0)
        return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: scales must be f32 or e8m0", name);
    if (c->pages < 0 || c->page_size < 1)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: invalid number or size of pages", name);
    if (c->pages > 0 && c->page_size > (int64_t(1) << 62) / c->pages)
        return b2k::fail(B2K_ERR_TOO_LARGE, "%s: too many slots", name);
    return B2K_OK;
}

int check_side(const b2k_pages &side, const b2k_heads &like, const b2k_cache &c, const char *name, const char *what,
               bool written) {
    if (side.heads != like.heads || (side.heads && side.dim != like.dim))
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: the %s cache has another number of heads or head size than %s", name,
                         what, what);
    if (side.heads == 0) return B2K_OK;
    if (side.group < 1 || side.dim % side.group || (side.group < 16 && side.group != side.dim))
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: the %s cache's scale group must be a head or a divisor of it >= 16",
                         name, what);
    if (c.pages == 0) return B2K_OK;
    if (side.codes_dev == nullptr || side.scales_dev == nullptr)
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: the %s cache holds a null pointer", name, what);
    if (c.scale_format == B2K_FMT_F32 && reinterpret_cast<uintptr_t>(side.scales_dev) % 4)
        return b2k::fail(B2K_ERR_ALIGNMENT, "%s: the %s cache's scales are not aligned to their items", name, what);
    const int64_t size[3] = {c.pages, c.page_size, side.heads};
    const int64_t codes[3] = {side.page_stride, side.slot_stride, side.head_stride};
    const int64_t scales[3] = {side.scale_page_stride, side.scale_slot_stride, side.scale_head_stride};
    if (written && (overlapping(3, size, codes, side.dim) || overlapping(3, size, scales, side.dim / side.group)))
        return b2k::fail(B2K_ERR_INVALID_ARG, "%s: rows of the %s cache overlap", name, what);
    return B2K_OK;
}

// ---- layout ----------------------------------------------------------------------------
// The stride of an axis of length 1 is never used: 0 keeps it out of the alignment rules.
void set_input(Role &r, const b2k_heads &h, int64_t tokens) {
    r.in = h.data_dev;
    r.in_token = tokens > 1 ? h.token_stride : 0;
    r.in_head = h.heads > 1 ? h.head_stride : 0;
    r.heads = static_cast<int>(h.heads);
    r.dim = static_cast<int>(h.dim);
    r.inv_dim = h.heads ? 1.0f / static_cast<float>(h.dim) : 0.0f;
}
void set_output(Role &r, const b2k_heads &h, int64_t tokens) {
    r.out = h.data_dev;
    r.out_token = tokens > 1 ? h.token_stride : 0;
    r.out_head = h.heads > 1 ? h.head_stride : 0;
}
void set_grad(Role &r, const b2k_heads &h, int64_t tokens) {
    r.grad = h.data_dev;
    r.grad_token = tokens > 1 ? h.token_stride : 0;
    r.grad_head = h.heads > 1 ? h.head_stride : 0;
}
void set_pages(Params &p, Role &r, const b2k_cache &c, const b2k_pages &side) {
    p.pages = c.pages;
    p.page_size = c.page_size;
    p.e5m2 = c.code_format == B2K_FMT_E5M2;
    p.e8m0 = c.scale_format == B2K_FMT_E8M0;
    r.codes = static_cast<uint8_t *>(side.codes_dev);
    r.scales = side.scales_dev;
    r.code_page = c.pages > 1 ? side.page_stride : 0;
    r.code_slot = c.page_size > 1 ? side.slot_stride : 0;
    r.code_head = side.heads > 1 ? side.head_stride : 0;
    r.scale_page = c.pages > 1 ? side.scale_page_stride : 0;
    r.scale_slot = c.page_size > 1 ? side.scale_slot_stride : 0;
    r.scale_head = side.heads > 1 ? side.scale_head_stride : 0;
    r.group = static_cast<int>(side.group);
}
void set_rotation(Params &p, const b2k_rotation &rot) {
    p.norm = static_cast<int>(rot.norm);
    p.eps = static_cast<float>(rot.eps);
    p.interleaved = static_cast<int>(rot.interleaved);
    p.weight_format = static_cast<int>(rot.weight_format);
    if (rot.norm) {
        p.role[0].weight = rot.q_weight_dev;
        p.role[1].weight = rot.k_weight_dev;
    }
    if (rot.rotary_dim > 0) {
        p.cos_table = rot.cos_dev;
        p.sin_table = rot.sin_dev;
        p.cos_stride = rot.table_rows > 1 ? rot.cos_stride : 0;
        p.sin_stride = rot.table_rows > 1 ? rot.sin_stride : 0;
    }
    if (has_positions(rot)) {
        p.table_rows = rot.table_rows;
        p.positions = rot.positions_dev;
        p.position_bytes = static_cast<int>(rot.position_bytes);
    }
}

static bool fits(const void *base, int64_t stride0, int64_t stride1, int itemsize, int vec) {
    return reinterpret_cast<uintptr_t>(base) % (static_cast<uintptr_t>(itemsize) * vec) == 0 && stride0 % vec == 0 &&
           stride1 % vec == 0;
}

// Whether every chunk of `vec` items of a role starts on a multiple of its size.
static bool role_fits(const Params &p, const Role &r, bool rotated, int rotary, int itemsize, int vec) {
    if (vec == 1) return true;
    if (r.dim % vec || !fits(r.in, r.in_token, r.in_head, itemsize, vec)) return false;
    if (r.out && !fits(r.out, r.out_token, r.out_head, itemsize, vec)) return false;
    if (r.grad && !fits(r.grad, r.grad_token, r.grad_head, itemsize, vec)) return false;
    if (r.weight && !fits(r.weight, 0, 0, item_bytes(p.weight_format), vec < 4 || p.weight_format != B2K_FMT_F32 ? vec : 4))
        return false;
    if (r.codes && (!fits(r.codes, r.code_page, r.code_slot, 1, vec) || r.code_head % vec || r.group % vec)) return false;
    if (rotated) {
        if (rotary % (p.interleaved ? vec : 2 * vec)) return false;
        const int w = vec / 2;                 // a chunk's pairs, or half a chunk of one table row
        if (!fits(p.cos_table, p.cos_stride, 0, 4, w) || !fits(p.sin_table, p.sin_stride, 0, 4, w)) return false;
    }
    return true;
}

// How chunks of `vec` items pair up in a role's rows; `turned` items are rotated.
static void pair_up(Role &r, int vec, int turned, bool interleaved) {
    // The halves of a rotated run pair up, and what lies behind it lies in pairs of
    // neighbouring chunks.  Without a rotation of halves the two halves of the row pair
    // up; single interleaved items (vec == 1) pair with their neighbours.
    if (turned && !interleaved) {
        r.pair_gap = turned / 2;
        r.tail = turned;
    } else if (turned && vec == 1) {
        r.pair_gap = r.tail = 0;
    } else {
        r.pair_gap = (r.dim / vec + 1) / 2 * vec;
        r.tail = r.dim;
    }
    r.pair_units = r.pair_gap / vec;
    r.angle_units = turned / 2 / vec;
    r.angle_items = turned;
    r.units = r.pair_units + (r.dim - r.tail + 2 * vec - 1) / (2 * vec);
}

// Units a lane holds in the smallest compiled shape for chunks of `vec` items; 0 if none
// takes so many.
static int units_a_lane(int vec, int units, int lanes) {
    const int need = (units + lanes - 1) / lanes;
#define B2K_HEADS_PICK(V, I) \
    if (vec == V && I >= need) return I;
    B2K_HEADS_SHAPES(B2K_HEADS_PICK)
#undef B2K_HEADS_PICK
    return 0;
}

int widest(const Params &p, int which, int64_t format, const b2k_rotation *rot) {
    const int itemsize = item_bytes(format);
    const int rotary = rot && which < 2 ? static_cast<int>(rot->rotary_dim) : 0;
    for (int vec : {8, 4, 2}) {
        if (vec * itemsize > 16 || !role_fits(p, p.role[which], rotary > 0, rotary, itemsize, vec)) continue;
        Role r = p.role[which];
        pair_up(r, vec, rotary, p.interleaved);
        if (units_a_lane(vec, r.units, 32)) return vec;
    }
    return 1;
}

Plan lay_out(Params &p, int vec, const b2k_rotation *rot) {
    Plan plan;
    plan.vec = vec;
    int units = 1;
    for (int i = 0; i < 3; ++i) {
        Role &r = p.role[i];
        if (r.heads == 0) continue;
        pair_up(r, vec, rot && i < 2 ? static_cast<int>(rot->rotary_dim) : 0, p.interleaved);
        if (r.units > units) units = r.units;
    }
    p.lanes = 1;
    p.lane_bits = 0;
    while (p.lanes < 32 && p.lanes < units) {
        p.lanes *= 2;
        p.lane_bits += 1;
    }
    plan.iter = units_a_lane(vec, units, p.lanes);
    // another role's narrow chunks may be too many for a long row: narrower ones have a shape
    if (plan.iter == 0 && vec > 1) return lay_out(p, vec / 2, rot);
    for (Role &r : p.role) {
        if (r.codes == nullptr) continue;
        r.groups_of = paging::divisor(static_cast<uint32_t>(r.group));
        // how the chunks of a scale's group lie over the lanes; see quantise_row
        const int span = r.group / plan.vec;
        const bool even = r.group % plan.vec == 0 && (span & (span - 1)) == 0;
        r.scale_lanes = 0;
        r.scale_joint = r.group == r.dim;
        if (r.scale_joint) r.scale_lanes = p.lanes;
        else if (plan.iter == 1 && even && r.tail == r.dim && r.dim == 2 * r.pair_gap && r.pair_gap % r.group == 0)
            r.scale_lanes = span;
    }
    return plan;
}

int count_items(Params &p, int most, int busy, const char *name) {
    // Several heads an item save loads of cosines, sines and weights and keep loads in
    // flight behind the arithmetic, but leave a small call with fewer groups than the GPU
    // has room for: halved until `busy` threads an SM have work.
    int64_t rows = 0;
    for (const Role &r : p.role) rows += r.heads;
    rows = rows > 0 && p.tokens > INT64_MAX / 64 / rows ? INT64_MAX / 64 : rows * p.tokens;
    while (most > 1 && rows * p.lanes / most < static_cast<int64_t>(busy) * b2k::sm_count()) most /= 2;
    const int64_t in_block = kThreads / p.lanes;
    int64_t blocks = 0;
    for (Role &r : p.role) {
        const int64_t per_token = (static_cast<int64_t>(r.heads) + most - 1) / most;
        r.heads_per_item = per_token ? static_cast<int>((r.heads + per_token - 1) / per_token) : 1;      // even shares
        if (per_token && p.tokens > INT_MAX / per_token)
            return b2k::fail(B2K_ERR_TOO_LARGE, "%s: more than 2^31 - 1 groups of rows", name);
        r.items = paging::divisor(static_cast<uint32_t>(per_token ? per_token : 1));
        r.all_items = static_cast<uint32_t>(p.tokens * per_token);
        r.blocks = static_cast<uint32_t>((p.tokens * per_token + in_block - 1) / in_block);
        blocks += r.blocks;
    }
    if (blocks > INT_MAX) return b2k::fail(B2K_ERR_TOO_LARGE, "%s: too many rows for one launch", name);
    return B2K_OK;
}

// ---- backward ----------------------------------------------------------------------------
// Blocks of a role stride over its rows and keep the weight gradient's partial sums in
// registers; each block writes one row of partials, and a second kernel adds the rows
// in order: no atomics, so equal calls give equal bits.
constexpr int kMostBlocksPerSm = 8;
constexpr int kBackwardHeadsPerItem = 8;
// 1024 tokens x 40 heads of 128 bf16 items: 15.7 us, with 512 18.5, with 2048 18.7.  Not measured
// for other types and heads.
constexpr int kBackwardBusy = 1024;

// The inverse rotation of a unit's pairs.
template <int FROM, int TO, int VEC>
__device__ __forceinline__ void turn_back(float (&x)[VEC], float (&y)[VEC], const float (&c)[VEC], const float (&s)[VEC]) {
    if constexpr (TO - FROM == 1) {
        const float u = x[FROM] * c[FROM] + y[FROM] * s[FROM], v = y[FROM] * c[FROM] - x[FROM] * s[FROM];
        x[FROM] = u;
        y[FROM] = v;
    } else {
#pragma unroll
        for (int j = FROM; j < TO; j += 2) {
            const float2 a = make_float2(x[j], x[j + 1]), b = make_float2(y[j], y[j + 1]);
            const float2 cc = make_float2(c[j], c[j + 1]), sn = make_float2(s[j], s[j + 1]);
            const float2 u = fma2(a, cc, mul2(b, sn));
            const float2 v = fma2(b, cc, mul2(make_float2(-a.x, -a.y), sn));
            x[j] = u.x;
            x[j + 1] = u.y;
            y[j] = v.x;
            y[j + 1] = v.y;
        }
    }
}

// sum of x^2 and of (g w) x over a chunk's worth of items, on top of ss and dot
template <int VEC>
__device__ __forceinline__ void gradient_sums(const float (&x)[VEC], const float (&g)[VEC], const float (&w)[VEC], float2 &ss,
                                              float2 &dot) {
    if constexpr (VEC == 1) {
        ss.x += x[0] * x[0];
        dot.x += g[0] * w[0] * x[0];
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 xx = make_float2(x[j], x[j + 1]);
            ss = fma2(xx, xx, ss);
            dot = fma2(mul2(make_float2(g[j], g[j + 1]), make_float2(w[j], w[j + 1])), xx, dot);
        }
    }
}

// g -> by (g w) - x pull, and the weight's sum += g x by
template <int VEC>
__device__ __forceinline__ void gradient_of(const float (&x)[VEC], float (&g)[VEC], const float (&w)[VEC], float by,
                                            float pull, float (&sum)[VEC]) {
    if constexpr (VEC == 1) {
        sum[0] += g[0] * (x[0] * by);
        g[0] = by * (g[0] * w[0]) - x[0] * pull;
    } else {
        const float2 by2 = make_float2(by, by), pull2 = make_float2(-pull, -pull);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 xx = make_float2(x[j], x[j + 1]), gg = make_float2(g[j], g[j + 1]);
            const float2 t = fma2(gg, mul2(xx, by2), make_float2(sum[j], sum[j + 1]));
            const float2 d = fma2(mul2(gg, make_float2(w[j], w[j + 1])), by2, mul2(xx, pull2));
            sum[j] = t.x;
            sum[j + 1] = t.y;
            g[j] = d.x;
            g[j + 1] = d.y;
        }
    }
}

// What a group knows of an item: its rows and where they start.
template <typename T>
struct Item {
    int64_t token;
    int rows;                    // 0 behind the last item
    const T *in, *grad;
    T *out;
    __device__ __forceinline__ void seek(const Role &r, uint32_t item) {
        const bool active = item < r.all_items;
        const uint32_t at_token = active ? r.items.quotient(item) : 0;
        token = at_token;
        const int first = active ? static_cast<int>(item - at_token * r.items.d) * r.heads_per_item : 0;
        rows = active ? min(r.heads - first, r.heads_per_item) : 0;
        in = static_cast<const T *>(r.in) + token * r.in_token + first * r.in_head;
        grad = static_cast<const T *>(r.grad) + token * r.grad_token + first * r.grad_head;
        out = static_cast<T *>(r.out) + token * r.out_token + first * r.out_head;
    }
};

// A lane's share of a role's weight and of its gradient, in the order of the pairs.
template <int VEC, int ITER>
struct Weights {
    float x[ITER][VEC], y[ITER][VEC], sum_x[ITER][VEC], sum_y[ITER][VEC];
};

// The gradient of one row as loaded (x and g, two chunks a unit), stored to `out` if `there`; a
// row that is not comes as zeros.
template <typename T, int VEC, int ITER, bool INTER, bool AHEAD>
__device__ __forceinline__ void gradient_row(const Params &p, const Role &r, const Lanes &g, const int (&oa)[ITER],
                                             const int (&ob)[ITER], const Chunk<T, VEC> (&xa)[ITER],
                                             const Chunk<T, VEC> (&xb)[ITER], const Chunk<T, VEC> (&da)[ITER],
                                             const Chunk<T, VEC> (&db)[ITER], const float (&c)[ITER][VEC],
                                             const float (&s)[ITER][VEC], Weights<VEC, ITER> &w, T *out, bool there) {
    float x[ITER][VEC], y[ITER][VEC], gx[ITER][VEC], gy[ITER][VEC];
    float2 ss = make_float2(0.0f, 0.0f), dot = ss;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        float a[VEC], b[VEC];
        widen(xa[i], a);
        widen(xb[i], b);
        in_pairs<VEC, INTER>(a, b, x[i], y[i]);
        widen(da[i], a);
        widen(db[i], b);
        in_pairs<VEC, INTER>(a, b, gx[i], gy[i]);
        const Turned t = turned_of<VEC, INTER>(r, g.lane + i * g.n, oa[i], ob[i]);
        if (VEC > 1 && t.lo) turn_back<0, VEC / 2, VEC>(gx[i], gy[i], c[i], s[i]);
        if (t.hi) turn_back<VEC / 2, VEC, VEC>(gx[i], gy[i], c[i], s[i]);
        gradient_sums<VEC>(x[i], gx[i], w.x[i], ss, dot);
        gradient_sums<VEC>(y[i], gy[i], w.y[i], ss, dot);
    }
    if (p.norm) {
        // dx = r (h - n mean(h n)) with n = x r:  r h - x (r^3 sum(h x) / dim)
        const float mean = g.sum(ss.x + ss.y) * r.inv_dim;
        const float by = !there ? 0.0f : rsqrtf(mean + p.eps);       // eps may be zero
        float pull = g.sum(dot.x + dot.y) * r.inv_dim * by * by * by;
        // Squares beyond float32: the result is zeros, and so is the gradient; but the sum of h x can
        // have passed the range too, and infinity times zero is no zero.  What is infinite or a NaN
        // itself still makes the row NaNs.  A group alone takes this branch where copies run ahead
        // (32768 tokens x 40 heads of 128 bf16 items: 170 us, with a vote of the warp 180), a warp
        // where registers are short (32 + 2 heads: 192 us, 217 for a group alone, which spills).
        const bool beyond = mean > FLT_MAX;
        if (AHEAD ? beyond : __any_sync(0xFFFFFFFFu, beyond)) {
            float none = 0.0f;
#pragma unroll
            for (int i = 0; i < ITER; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) none += x[i][j] * 0.0f + y[i][j] * 0.0f;
            none = AHEAD ? g.sum_alone(none) : g.sum(none);
            if (beyond) pull = none;
        }
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            gradient_of<VEC>(x[i], gx[i], w.x[i], by, pull, w.sum_x[i]);
            gradient_of<VEC>(y[i], gy[i], w.y[i], by, pull, w.sum_y[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        float a[VEC], b[VEC];
        out_of_pairs<VEC, INTER>(gx[i], gy[i], a, b);
        if (there && oa[i] < r.dim) store_chunk<T, VEC>(out + oa[i], a);
        if (there && ob[i] < r.dim) store_chunk<T, VEC>(out + ob[i], b);
    }
}

// A padding token's row: not computed, since a weight's infinity times zero is no zero.
template <typename T, int VEC, int ITER>
__device__ __forceinline__ void zero_row(T *out, const int (&oa)[ITER], const int (&ob)[ITER], int dim) {
    const float zeros[VEC] = {};
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (oa[i] < dim) store_chunk<T, VEC>(out + oa[i], zeros);
        if (ob[i] < dim) store_chunk<T, VEC>(out + ob[i], zeros);
    }
}

__device__ __forceinline__ bool is_padding(const Params &p, int64_t position) {
    return p.positions != nullptr && (position < 0 || position >= p.table_rows);
}
__device__ __forceinline__ int64_t position_of(const Params &p, int64_t token) {
    return p.positions != nullptr ? paging::load_index(p.positions, p.position_bytes, token) : 0;
}

// The rows of a warp's items `base`, `base + step`, ..., the next row loaded into registers
// while one is worked on.  A warp's groups take neighbouring items and stay together: see
// Lanes.  all_items < 2^31, and a step is at most the grid's groups, so nothing overflows.
template <typename T, int VEC, int ITER, bool INTER>
__device__ __forceinline__ void backward_rows(const Params &p, const Role &r, const Lanes &g, uint32_t base, uint32_t step,
                                              const int (&oa)[ITER], const int (&ob)[ITER], Weights<VEC, ITER> &w) {
    for (; base < r.all_items; base += step) {
        Item<T> it;
        it.seek(r, base + (threadIdx.x % 32 >> p.lane_bits));
        Batch<T, VEC, ITER, 1> x_now, g_now;
        x_now.load(it.in, 0, it.rows, oa, ob, r.dim);
        g_now.load(it.grad, 0, it.rows, oa, ob, r.dim);
        const int64_t position = position_of(p, it.token);
        const bool padding = is_padding(p, position);
        if (padding) {
            x_now = Batch<T, VEC, ITER, 1>{};
            g_now = Batch<T, VEC, ITER, 1>{};
        }
        const int loads = padding ? 0 : it.rows;
        float c[ITER][VEC], s[ITER][VEC];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int u = g.lane + i * g.n;
            Turned t = turned_of<VEC, INTER>(r, u, oa[i], ob[i]);
            t.lo = t.lo && !padding;
            t.hi = t.hi && !padding;
            load_angles<VEC, INTER>(p.cos_table + position * p.cos_stride, u, oa[i], ob[i], t, c[i]);
            load_angles<VEC, INTER>(p.sin_table + position * p.sin_stride, u, oa[i], ob[i], t, s[i]);
        }
        const int most = __reduce_max_sync(0xFFFFFFFFu, it.rows);
#pragma unroll 1
        for (int h = 0; h < most; ++h) {
            Batch<T, VEC, ITER, 1> x_next, g_next;
            it.in += r.in_head;
            it.grad += r.grad_head;
            x_next.load(it.in, 0, loads - h - 1, oa, ob, r.dim);
            g_next.load(it.grad, 0, loads - h - 1, oa, ob, r.dim);
            gradient_row<T, VEC, ITER, INTER, false>(p, r, g, oa, ob, x_now.a[0], x_now.b[0], g_now.a[0], g_now.b[0], c, s, w, it.out,
                                                     !padding && h < it.rows);
            if (padding && h < it.rows) zero_row<T, VEC, ITER>(it.out, oa, ob, r.dim);
            it.out += r.out_head;
            x_now = x_next;
            g_now = g_next;
        }
    }
}

// The same with the rows of kStages - 1 steps ahead on their way into shared memory, across
// the ends of items, with the next item's cosines and sines: registers no longer limit
// the bytes in flight, and no warp waits for a position and then for its table rows.
// Every thread copies what it will read itself, so there is nothing to synchronise but its
// own copies.  32768 tokens x 40 heads of 128 bf16 items, three sets of inputs in turn: 198 us
// with the next row in registers, 172 us so, 177 us with four stages.  Needs 16-byte chunks, one unit a lane,
// and items of at least kStages steps (then the loads are at most one item ahead).
constexpr int kStages = 3;

template <int VEC>
struct Ring {
    static constexpr int half = VEC * 2;             // bytes of VEC / 2 floats
    static constexpr int rows = kStages * 4 * kThreads * 16, tables = 2 * 4 * kThreads * half;
};

// Shared memory of a block: the copies, and later one row of floats per warp for the
// weight's sums (rows of one unit a lane have at most 64 * VEC items).
template <typename T, int VEC, bool AHEAD>
constexpr int shared_bytes() {
    return AHEAD ? Ring<VEC>::rows + Ring<VEC>::tables : kThreads / 32 * B2K_MAX_HEAD_DIM * 4;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void *to_shared, const void *from) {
    const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(to_shared));
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void backward_rows_ahead(const Params &p, const Role &r, const Lanes &g, uint32_t base, uint32_t step,
                                                    const int (&oa)[1], const int (&ob)[1], Weights<VEC, 1> &w, char *shared) {
    using Slots = Ring<VEC>;
    constexpr int H = VEC / 2;
    const int hpi = r.heads_per_item;
    const uint32_t in_warp = threadIdx.x % 32 >> p.lane_bits;
    const Turned turned = turned_of<VEC, INTER>(r, g.lane, oa[0], ob[0]);
    const int at_lo = INTER ? oa[0] / 2 : g.lane * VEC, at_hi = INTER ? ob[0] / 2 : g.lane * VEC + H;
    const bool has_a = oa[0] < r.dim, has_b = ob[0] < r.dim;
    // slots are [stage][array][thread], so neighbouring threads' 16 bytes are neighbours
    char *const row_slot = shared + threadIdx.x * 16;
    char *const table_slot = shared + Slots::rows + threadIdx.x * Slots::half;

    if (base >= r.all_items) return;
    // the load side: its item, row and position, and the position of the item after it
    Item<T> ahead;
    ahead.seek(r, base + in_warp);
    uint32_t ahead_base = base;
    int ahead_h = 0, ahead_stage = 0, ahead_table = 0;
    int64_t ahead_position = 0, after_position = 0;
    const auto later_position = [&](uint32_t at) {
        const uint32_t item = at + in_warp;
        return item < r.all_items ? position_of(p, r.items.quotient(item)) : 0;
    };
    const auto load_step = [&]() {
        if (ahead_base < r.all_items) {
            if (ahead_h == 0 && p.positions != nullptr && !is_padding(p, ahead_position) && ahead.rows > 0) {
                char *to = table_slot + ahead_table * 4 * kThreads * Slots::half;
                const float *c = p.cos_table + ahead_position * p.cos_stride, *s = p.sin_table + ahead_position * p.sin_stride;
                if (turned.lo) {
                    copy_async<Slots::half>(to, c + at_lo);
                    copy_async<Slots::half>(to + 2 * kThreads * Slots::half, s + at_lo);
                }
                if (turned.hi) {
                    copy_async<Slots::half>(to + kThreads * Slots::half, c + at_hi);
                    copy_async<Slots::half>(to + 3 * kThreads * Slots::half, s + at_hi);
                }
            }
            if (ahead_h < ahead.rows) {
                char *to = row_slot + ahead_stage * 4 * kThreads * 16;
                if (has_a) {
                    copy_async<16>(to, ahead.in + oa[0]);
                    copy_async<16>(to + 2 * kThreads * 16, ahead.grad + oa[0]);
                }
                if (has_b) {
                    copy_async<16>(to + kThreads * 16, ahead.in + ob[0]);
                    copy_async<16>(to + 3 * kThreads * 16, ahead.grad + ob[0]);
                }
            }
            ahead.in += r.in_head;
            ahead.grad += r.grad_head;
            if (++ahead_h == hpi) {
                ahead_h = 0;
                ahead_table ^= 1;
                ahead_base += step;
                ahead.seek(r, ahead_base + in_warp);
                ahead_position = after_position;
                after_position = later_position(ahead_base + step);
            }
        }
        commit_copies();
        ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
    };

    ahead_position = later_position(base);
    after_position = later_position(base + step);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) load_step();

    int stage = 0, table = 0;
    for (; base < r.all_items; base += step) {
        // the load side is still in this item: see kStages
        const int rows = ahead.rows;
        T *out = ahead.out;
        const bool padding = is_padding(p, ahead_position);
#pragma unroll 1
        for (int h = 0; h < hpi; ++h) {
            wait_copies<kStages - 2>();
            // read again for every row: 16 registers less
            float c[1][VEC], s[1][VEC];
            const char *angles = table_slot + table * 4 * kThreads * Slots::half;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                float cc[H], ss[H];
                load_floats<H>(reinterpret_cast<const float *>(angles + part * kThreads * Slots::half), cc);
                load_floats<H>(reinterpret_cast<const float *>(angles + (2 + part) * kThreads * Slots::half), ss);
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    c[0][part * H + i] = cc[i];
                    s[0][part * H + i] = ss[i];
                }
            }
            const T *from = reinterpret_cast<const T *>(row_slot + stage * 4 * kThreads * 16);
            constexpr int next = kThreads * 16 / sizeof(T);
            const bool there = h < rows;
            Chunk<T, VEC> xa[1], xb[1], da[1], db[1];
            xa[0] = load_chunk<T, VEC>(from);
            xb[0] = load_chunk<T, VEC>(from + next);
            da[0] = load_chunk<T, VEC>(from + 2 * next);
            db[0] = load_chunk<T, VEC>(from + 3 * next);
            // What no copy has filled, angles too, holds anything: zeros instead.  One vote for
            // the common row, where there is nothing of the kind, in place of a select for
            // every register.
            const bool row = there && !padding;
            if (__any_sync(0xFFFFFFFFu, !(row && has_a && has_b))) {
                if (!(row && has_a)) xa[0] = da[0] = Chunk<T, VEC>{};
                if (!(row && has_b)) xb[0] = db[0] = Chunk<T, VEC>{};
                if (!row)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) c[0][j] = s[0][j] = 0.0f;
                if (there && padding) zero_row<T, VEC, 1>(out, oa, ob, r.dim);
            }
            load_step();                     // into the slot that the step before this one read
            gradient_row<T, VEC, 1, INTER, true>(p, r, g, oa, ob, xa, xb, da, db, c, s, w, out, row);
            out += r.out_head;
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        table ^= 1;
    }
    wait_copies<0>();
}

template <typename T, int VEC, int ITER, bool AHEAD, int WHICH, bool INTER>
__device__ __forceinline__ void backward_role(const Params &p, uint32_t first_block, uint32_t blocks, char *shared) {
    const Role &r = p.role[WHICH];
    const Lanes g(p.lanes);
    const uint32_t in_block = static_cast<uint32_t>(kThreads) >> p.lane_bits;
    int oa[ITER], ob[ITER];
    Weights<VEC, ITER> w;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        unit_at<VEC>(r, g.lane + i * g.n, oa[i], ob[i]);
        float wa[VEC] = {}, wb[VEC] = {};
        if (oa[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, oa[i], wa);
        if (ob[i] < r.dim) load_weight<VEC>(r.weight, p.weight_format, ob[i], wb);
        in_pairs<VEC, INTER>(wa, wb, w.x[i], w.y[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) w.sum_x[i][j] = w.sum_y[i][j] = 0.0f;
    }
    const uint32_t base = first_block * in_block + threadIdx.x / 32 * (32u >> p.lane_bits), step = blocks * in_block;
    if constexpr (AHEAD) backward_rows_ahead<T, VEC, INTER>(p, r, g, base, step, oa, ob, w, shared);
    else backward_rows<T, VEC, ITER, INTER>(p, r, g, base, step, oa, ob, w);
    if (r.weight_grad == nullptr) return;
    // groups of a warp, then the block's warps in order
    __syncthreads();                                     // the copies' memory is free now
    float *block_sums = reinterpret_cast<float *>(shared);       // one row of dim floats per warp
    const int warp = threadIdx.x / 32;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        float a[VEC], b[VEC];
        out_of_pairs<VEC, INTER>(w.sum_x[i], w.sum_y[i], a, b);
        for (int o = g.n; o < 32; o *= 2)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                a[j] += __shfl_xor_sync(0xFFFFFFFFu, a[j], o);
                b[j] += __shfl_xor_sync(0xFFFFFFFFu, b[j], o);
            }
        if (threadIdx.x % 32 < g.n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (oa[i] < r.dim) block_sums[warp * r.dim + oa[i] + j] = a[j];
                if (ob[i] < r.dim) block_sums[warp * r.dim + ob[i] + j] = b[j];
            }
        }
    }
    __syncthreads();
    float *row = p.partials + static_cast<int64_t>(blockIdx.x) * p.partial_stride;
    for (int d = threadIdx.x; d < r.dim; d += kThreads) {
        float v = 0.0f;
        for (int k = 0; k < kThreads / 32; ++k) v += block_sums[k * r.dim + d];
        row[d] = v;
    }
}

// Four blocks an SM where a row takes one unit a lane (128 registers; 32768 tokens x 40
// heads of 128 bf16 items, three sets of inputs in turn: 172 us, with three blocks 178 us).
template <typename T, int VEC, int ITER, bool AHEAD>
__global__ void __launch_bounds__(kThreads, ITER == 1 ? 4 : 1) heads_backward_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(16) char shared[];
    const uint32_t blocks0 = p.blocks0, blocks1 = gridDim.x - blocks0;
    if (VEC > 1 && p.interleaved) {
        if (blockIdx.x < blocks0) backward_role<T, VEC, ITER, AHEAD, 0, true>(p, blockIdx.x, blocks0, shared);
        else backward_role<T, VEC, ITER, AHEAD, 1, true>(p, blockIdx.x - blocks0, blocks1, shared);
    } else {
        if (blockIdx.x < blocks0) backward_role<T, VEC, ITER, AHEAD, 0, false>(p, blockIdx.x, blocks0, shared);
        else backward_role<T, VEC, ITER, AHEAD, 1, false>(p, blockIdx.x - blocks0, blocks1, shared);
    }
}

// weight_grad[d] = sum over the role's blocks of partials[block][d], 32 columns a block: 32
// warps stride over the partial rows with four loads in flight, then one warp a column
// folds their sums.  The order depends on the grid alone.  (With 4 warps and one load in
// flight this took 25 us for 592 rows of 128.)
constexpr int kSumThreads = 1024;

__global__ void __launch_bounds__(kSumThreads) weight_grad_kernel(const __grid_constant__ Params p, int blocks) {
    __shared__ float part[32][33];
    const Role &r = p.role[blockIdx.y];
    if (r.weight_grad == nullptr) return;
    const int column = threadIdx.x % 32, row = threadIdx.x / 32;
    const int begin = blockIdx.y ? p.blocks0 : 0, end = blockIdx.y ? blocks : p.blocks0;
    const int d = blockIdx.x * 32 + column;
    float v[4] = {};
    if (d < r.dim)
        for (int b = begin + row; b < end; b += 4 * 32)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (b + i * 32 < end) v[i] += p.partials[static_cast<int64_t>(b + i * 32) * p.partial_stride + d];
    part[row][column] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    float sum = part[column][row];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const int at = blockIdx.x * 32 + row;
    if (column || at >= r.dim) return;
    if (p.weight_format == B2K_FMT_F32) static_cast<float *>(r.weight_grad)[at] = sum;
    else if (p.weight_format == B2K_FMT_F16) static_cast<__half *>(r.weight_grad)[at] = __float2half_rn(sum);
    else static_cast<__nv_bfloat16 *>(r.weight_grad)[at] = __float2bfloat16_rn(sum);
}

// Blocks of one instantiation that an SM holds at once: the grid is at most one wave, since
// a second, partial one would leave most SMs idle (4 blocks an SM where 3 fit cost 40%).
template <typename T, int VEC, int ITER, bool AHEAD>
int resident_blocks() {
    static b2k::PerDeviceOnce once;
    static int found[b2k::kMaxDevices];
    const int dev = b2k::current_device();
    if (dev < 0 || dev >= b2k::kMaxDevices) return 1;
    once.run([&] {
        int n = 0;
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(
            &n, heads_backward_kernel<T, VEC, ITER, AHEAD>, kThreads, shared_bytes<T, VEC, AHEAD>());
        found[dev] = n < 1 ? 1 : n > kMostBlocksPerSm ? kMostBlocksPerSm : n;
        return e;
    });
    return found[dev] < 1 ? 1 : found[dev];
}

// Launches `blocks` blocks, or with none says how many an SM holds.
template <typename T, int VEC, int ITER, bool AHEAD>
int backward_shape(const Params &p, int blocks, cudaStream_t stream) {
    if (blocks == 0) return resident_blocks<T, VEC, ITER, AHEAD>();
    heads_backward_kernel<T, VEC, ITER, AHEAD><<<blocks, kThreads, shared_bytes<T, VEC, AHEAD>(), stream>>>(p);
    return 0;
}

template <typename T>
static int pick_backward(const Params &p, const Plan &plan, int blocks, cudaStream_t stream) {
    // copies ahead need items of at least kStages steps in every role
    bool ahead = true;
    for (const Role &r : p.role) ahead = ahead && (r.heads == 0 || r.heads_per_item >= kStages);
#define B2K_HEADS_CASE(V, I)                                                                              \
    if constexpr (V * sizeof(T) <= 16)                                                                    \
        if (plan.vec == V && plan.iter == I) {                                                            \
            if constexpr (V * sizeof(T) == 16 && I == 1)                                                  \
                if (ahead) return backward_shape<T, V, I, true>(p, blocks, stream);                       \
            return backward_shape<T, V, I, false>(p, blocks, stream);                                     \
        }
    B2K_HEADS_SHAPES(B2K_HEADS_CASE)
#undef B2K_HEADS_CASE
    return 1;
}

static int backward_kernel(int64_t format, const Params &p, const Plan &plan, int blocks, cudaStream_t stream) {
    if (format == B2K_FMT_F32) return pick_backward<float>(p, plan, blocks, stream);
    if (format == B2K_FMT_F16) return pick_backward<__half>(p, plan, blocks, stream);
    return pick_backward<__nv_bfloat16>(p, plan, blocks, stream);
}

}  // namespace headwise

extern "C" {

using namespace headwise;

int b2k_norm_rotate(const b2k_rotation *r, const b2k_heads *q_out, const b2k_heads *k_out, void *stream) {
    B2K_RANGE("b2k_norm_rotate");
    const char *name = "b2k_norm_rotate";
    if (int rc = check_rotation(r, name)) return rc;
    if (q_out == nullptr || k_out == nullptr) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    Params p{};
    const b2k_heads *in[2] = {&r->q, &r->k}, *out[2] = {q_out, k_out};
    for (int i = 0; i < 2; ++i) {
        const char *what = i ? "k_out" : "q_out";
        if (int rc = check_heads(*out[i], name, what, r->tokens, item_bytes(r->format), true)) return rc;
        if (int rc = check_like(*out[i], *in[i], name, what)) return rc;
        if (in[i]->heads == 0) continue;
        set_input(p.role[i], *in[i], r->tokens);
        set_output(p.role[i], *out[i], r->tokens);
    }
    if (r->tokens == 0) return B2K_OK;
    p.tokens = r->tokens;
    set_rotation(p, *r);
    return launch_forward<kRotate>(p, r->format, r, b2k::as_stream(stream), name);
}

int64_t b2k_norm_rotate_backward_scratch_bytes(const b2k_rotation *r) {
    const int64_t dim = r == nullptr || (r->q.heads == 0 && r->k.heads == 0) ? B2K_MAX_HEAD_DIM
                        : r->k.heads == 0 || (r->q.heads && r->q.dim > r->k.dim) ? r->q.dim : r->k.dim;
    if (dim < 0 || dim > B2K_MAX_HEAD_DIM) return 0;
    return static_cast<int64_t>(b2k::sm_count()) * kMostBlocksPerSm * dim * 4;
}

int b2k_norm_rotate_backward(const b2k_rotation *r, const b2k_heads *q_grad, const b2k_heads *k_grad,
                             const b2k_heads *dq, const b2k_heads *dk, void *dq_weight_dev, void *dk_weight_dev,
                             void *scratch_dev, int64_t scratch_bytes, void *stream) {
    B2K_RANGE("b2k_norm_rotate_backward");
    const char *name = "b2k_norm_rotate_backward";
    if (int rc = check_rotation(r, name)) return rc;
    if (!q_grad || !k_grad || !dq || !dk) return b2k::fail(B2K_ERR_INVALID_ARG, "%s: null arguments", name);
    Params p{};
    const b2k_heads *in[2] = {&r->q, &r->k}, *grad[2] = {q_grad, k_grad}, *out[2] = {dq, dk};
    void *weight_grad[2] = {dq_weight_dev, dk_weight_dev};
    const int itemsize = item_bytes(r->format);
    for (int i = 0; i < 2; ++i) {
        if (int rc = check_heads(*grad[i], name, i ? "k_grad" : "q_grad", r->tokens, itemsize, false)) return rc;
        if (int rc = check_heads(*out[i], name, i ? "dk" : "dq", r->tokens, itemsize, true)) return rc;
        if (int rc = check_like(*grad[i], *in[i], name, i ? "k_grad" : "q_grad")) return rc;
        if (int rc = check_like(*out[i], *in[i], name, i ? "dk" : "dq")) return rc;
        if (weight_grad[i]) {
            const void *w = i ? r->k_weight_dev : r->q_weight_dev;
            if (!r->norm || in[i]->heads == 0 || w == nullptr)
                return b2k::fail(B2K_ERR_INVALID_ARG, "%s: the gradient of a weight that is not there is asked for", name);
            if (reinterpret_cast<uintptr_t>(weight_grad[i]) % item_bytes(r->weight_format))
                return b2k::fail(B2K_ERR_ALIGNMENT, "%s: a weight's gradient is not aligned to its items", name);
        }
        if (in[i]->heads == 0) continue;
        set_input(p.role[i], *in[i], r->tokens);
        set_grad(p.role[i], *grad[i], r->tokens);
        set_output(p.role[i], *out[i], r->tokens);
        p.role[i].weight_grad = weight_grad[i];
    }
    const bool summed = dq_weight_dev || dk_weight_dev;
    if (r->tokens == 0 && !summed) return B2K_OK;
    if (summed && (scratch_dev == nullptr || scratch_bytes < b2k_norm_rotate_backward_scratch_bytes(r)))
        return b2k::fail(B2K_ERR_SCRATCH, "%s: scratch is missing or too small", name);
    if (reinterpret_cast<uintptr_t>(scratch_dev) % 4)
        return b2k::fail(B2K_ERR_ALIGNMENT, "%s: scratch is not aligned", name);
    p.tokens = r->tokens;
    p.partials = static_cast<float *>(scratch_dev);
    set_rotation(p, *r);
    int vec = 8;
    for (int i = 0; i < 2; ++i)
        if (p.role[i].heads) vec = std::min(vec, widest(p, i, r->format, r));
    const Plan plan = lay_out(p, vec, r);
    if (plan.iter == 0) return b2k::fail(B2K_ERR_UNSUPPORTED, "%s: no kernel for this head size", name);
    if (int rc = count_items(p, kBackwardHeadsPerItem, kBackwardBusy, name)) return rc;
    if (r->tokens > 0)
        if (int rc = check_apart(p.role[0].out, p.role[1].out, name, "dq and dk")) return rc;
    if (int rc = check_apart(dq_weight_dev, dk_weight_dev, name, "the weights' gradients")) return rc;
    const cudaStream_t st = b2k::as_stream(stream);
    const int64_t most = b2k::sm_count() * static_cast<int64_t>(backward_kernel(r->format, p, plan, 0, st));
    int64_t need[2] = {p.role[0].blocks, p.role[1].blocks};
    // one wave, and as many blocks as give each the same number of rounds: 2.2 rounds of a
    // full wave take as long as 3 (4096 tokens x 40 heads of 128 bf16 items: 41 us)
    for (int64_t rounds = std::max<int64_t>(1, (need[0] + need[1] + most - 1) / most);; ++rounds) {
        const int64_t share[2] = {(need[0] + rounds - 1) / rounds, (need[1] + rounds - 1) / rounds};
        if (share[0] + share[1] > most) continue;
        need[0] = share[0];
        need[1] = share[1];
        break;
    }
    p.blocks0 = static_cast<int>(need[0]);
    const int blocks = static_cast<int>(need[0] + need[1]);
    const int dim = p.role[0].dim > p.role[1].dim ? p.role[0].dim : p.role[1].dim;
    p.partial_stride = dim;
    if (blocks > 0) {
        backward_kernel(r->format, p, plan, blocks, st);
        B2K_RETURN_IF_LAUNCH_FAILED(name);
        b2k::note_launch();
    }
    if (summed) {
        weight_grad_kernel<<<dim3((dim + 31) / 32, 2), kSumThreads, 0, st>>>(p, blocks);
        B2K_RETURN_IF_LAUNCH_FAILED(name);
        b2k::note_launch();
    }
    return B2K_OK;
}

}  // extern "C"
