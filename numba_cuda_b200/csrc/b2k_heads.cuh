// Row arithmetic shared by the head-wise kernels (b2k_headnorm.cu, b2k_kvcache.cu).
//
// A row is one head of one token, dim <= 1024 items.  It is owned by a group of 1..32
// lanes of one warp; a lane owns `units` of the row, each a pair of chunks of VEC items.
// The two chunks of a unit are chosen so that every rotated pair (i, i + R/2) lies in
// ONE lane: the rotation needs no exchange between lanes, and neighbouring lanes still
// read neighbouring chunks.  The row stays in registers from its load to its store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "b2k_internal.cuh"
#include "b2k_pages.cuh"

namespace headwise {

constexpr int kThreads = 128;

// Rows of one token that a group has in flight at once, and in all: cosines, sines and
// weights are loaded once for the latter.  Rows that spread over several units a lane
// leave registers for one.
B2K_HD constexpr int rows_in_flight(int iter) { return iter == 1 ? 2 : 1; }
constexpr int kHeadsPerItem = 16;

// One array role of a launch (queries, keys or values).
struct Role {
    const void *in;
    void *out;                  // null: the role is quantised into the cache
    const void *grad;           // backward: the gradient of the role's output
    int64_t in_token, in_head, out_token, out_head, grad_token, grad_head;
    const void *weight;
    void *weight_grad;
    uint8_t *codes;
    void *scales;
    int64_t code_page, code_slot, code_head, scale_page, scale_slot, scale_head;
    int heads, dim, group;
    paging::Divisor items;              // items of work a token has in this role: ceil(heads / heads_per_item)
    paging::Divisor groups_of;          // division by `group`
    uint32_t all_items, blocks; // of the launch
    int units;                  // chunk pairs of a row
    int pair_units, pair_gap, tail;   // units below pair_units are (u, u + gap); the others lie from `tail` on
    int angle_units;            // units below it are rotated (pairs of halves, or of single items)
    int angle_items;            // chunks below it are rotated (interleaved pairs)
    int heads_per_item;
    int scale_lanes, scale_joint;     // lanes that share a scale (0: found through shared memory), and whether
                                      // a lane's two chunks do
    float inv_dim;
};

struct Params {
    Role role[3];
    int64_t tokens;
    int lanes, lane_bits;
    int norm, interleaved, weight_format;
    float eps;
    const float *cos_table, *sin_table;
    int64_t cos_stride, sin_stride, table_rows;
    const void *positions;
    int position_bytes;
    const void *slots;
    int slot_bytes, e5m2, e8m0;
    int64_t pages, page_size;
    float *partials;            // backward: weight-gradient partial sums, a row per block
    int partial_stride;
    int blocks0;                // backward: blocks of role 0
};

// Moves go by whole words: 1, 2, 4, 8 or 16 bytes as one access.
template <int BYTES> struct WordOf;
template <> struct WordOf<1> { using type = uint8_t; };
template <> struct WordOf<2> { using type = uint16_t; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<16> { using type = uint4; };

// VEC items of type T as loaded.
template <typename T, int VEC>
union Chunk {
    using Word = typename WordOf<sizeof(T) * VEC>::type;
    Word all;
    uint32_t word[sizeof(T) * VEC < 4 ? 1 : sizeof(T) * VEC / 4];
};

template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T *p) {
    Chunk<T, VEC> c;
    c.all = *reinterpret_cast<const typename Chunk<T, VEC>::Word *>(p);
    return c;
}

__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<const uint32_t *>(&v); }
__device__ __forceinline__ uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t *>(&v); }

// float32 <-> T.  A bfloat16 is the upper half of a float32, so it is widened by a shift
// or a mask.
template <typename T> struct Convert;
template <> struct Convert<float> {
    __device__ static float down(float x) { return x; }
};
template <> struct Convert<__half> {
    __device__ static float2 up2(uint32_t two) { return __half22float2(*reinterpret_cast<const __half2 *>(&two)); }
    __device__ static __half down(float x) { return __float2half_rn(x); }
    __device__ static uint32_t down2(float lo, float hi) { return bits(__floats2half2_rn(lo, hi)); }
};
template <> struct Convert<__nv_bfloat16> {
    __device__ static float2 up2(uint32_t two) {
        return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xFFFF0000u));
    }
    __device__ static __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
    __device__ static uint32_t down2(float lo, float hi) { return bits(__floats2bfloat162_rn(lo, hi)); }
};

template <typename T, int VEC>
__device__ __forceinline__ void widen(const Chunk<T, VEC> &c, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = __uint_as_float(c.word[j]);
    } else if constexpr (VEC == 1) {
        v[0] = Convert<T>::up2(c.all).x;
    } else {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            const float2 f = Convert<T>::up2(c.word[j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        *p = Convert<T>::down(v[0]);
    } else {
        Chunk<T, VEC> c;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) c.word[j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) c.word[j] = Convert<T>::down2(v[2 * j], v[2 * j + 1]);
        }
        *reinterpret_cast<typename Chunk<T, VEC>::Word *>(p) = c.all;
    }
}

// Two float32 operations in one instruction (sm_100).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; "
        "mov.b64 {%0, %1}, x;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

template <int VEC>
__device__ __forceinline__ void load_floats(const float *p, float (&v)[VEC]) {
    constexpr int W = VEC < 4 ? VEC : 4;       // 16 bytes at most
#pragma unroll
    for (int j = 0; j < VEC; j += W) {
        const Chunk<float, W> c = load_chunk<float, W>(p + j);
#pragma unroll
        for (int i = 0; i < W; ++i) v[j + i] = __uint_as_float(c.word[i]);
    }
}

template <int VEC>
__device__ __forceinline__ void load_weight(const void *w, int format, int at, float (&v)[VEC]) {
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 1.0f;
    } else if (format == B2K_FMT_F32) {
        load_floats<VEC>(static_cast<const float *>(w) + at, v);
    } else if (format == B2K_FMT_BF16) {
        widen(load_chunk<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16 *>(w) + at), v);
    } else {
        widen(load_chunk<__half, VEC>(static_cast<const __half *>(w) + at), v);
    }
}

// The lanes of a group.  Reductions are called by whole warps, idle groups included: a
// shuffle under a mask known only at run time costs a warp synchronisation each, which
// is what bounded the kernels that let idle groups leave early.
struct Lanes {
    int n, lane;
    __device__ explicit Lanes(int lanes) : n(lanes), lane(threadIdx.x & (lanes - 1)) {}
    __device__ float sum(float v) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o < n) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        return v;
    }
    // for a group that is alone in a branch
    __device__ float sum_alone(float v) const {
        const unsigned group = (0xFFFFFFFFu >> (32 - n)) << (threadIdx.x & 31 & ~(n - 1));
        for (int o = n / 2; o > 0; o >>= 1) v += __shfl_xor_sync(group, v, o);
        return v;
    }
    // over aligned runs of `span` lanes (a power of two) of the group
    __device__ float max(float v, int span) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o < span) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
        return v;
    }
};

// Where a unit's two chunks start.
template <int VEC>
__device__ __forceinline__ void unit_at(const Role &r, int u, int &a, int &b) {
    if (u < r.pair_units) {
        a = u * VEC;
        b = a + r.pair_gap;
    } else {
        a = r.tail + 2 * (u - r.pair_units) * VEC;
        b = a + VEC;
    }
    if (u >= r.units) a = b = r.dim;       // nothing
}

// A group's chunks of ROWS rows of one token, as loaded.
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

// Items of a chunk pair as they meet in a rotation: pair j of a unit is (a[j], b[j]), or
// neighbouring items of one chunk when interleaved (VEC == 1: always the unit's two
// items).  `pair` copies the items into that order and `unpair` back; the copies are
// register names, not instructions.
template <int VEC>
__device__ __forceinline__ void pair(const float (&a)[VEC], const float (&b)[VEC], float (&x)[VEC], float (&y)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float *from = 2 * j < VEC ? a : b;
        const int at = 2 * j < VEC ? 2 * j : 2 * j - VEC;
        x[j] = VEC == 1 ? a[0] : from[at];
        y[j] = VEC == 1 ? b[0] : from[at + (VEC > 1)];
    }
}
template <int VEC>
__device__ __forceinline__ void unpair(const float (&x)[VEC], const float (&y)[VEC], float (&a)[VEC], float (&b)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        float *to = 2 * j < VEC ? a : b;
        const int at = 2 * j < VEC ? 2 * j : 2 * j - VEC;
        if (VEC == 1) {
            a[0] = x[0];
            b[0] = y[0];
        } else {
            to[at] = x[j];
            to[at + (VEC > 1)] = y[j];
        }
    }
}

// INTER is a constant because a choice at run time costs a move per item.
template <int VEC, bool INTER>
__device__ __forceinline__ void in_pairs(const float (&a)[VEC], const float (&b)[VEC], float (&x)[VEC], float (&y)[VEC]) {
    if constexpr (INTER) {
        pair<VEC>(a, b, x, y);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            x[j] = a[j];
            y[j] = b[j];
        }
    }
}
template <int VEC, bool INTER>
__device__ __forceinline__ void out_of_pairs(const float (&x)[VEC], const float (&y)[VEC], float (&a)[VEC], float (&b)[VEC]) {
    if constexpr (INTER) {
        unpair<VEC>(x, y, a, b);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            a[j] = x[j];
            b[j] = y[j];
        }
    }
}

// Which half of a unit's pairs is rotated: all or none for pairs of halves, one chunk's
// pairs each when interleaved.
struct Turned {
    bool lo, hi;
};
template <int VEC, bool INTER>
__device__ __forceinline__ Turned turned_of(const Role &r, int u, int oa, int ob) {
    if (VEC > 1 && INTER) return Turned{oa < r.angle_items, ob < r.angle_items};
    return Turned{u < r.angle_units, u < r.angle_units};
}

// A unit's cosines or sines, from its position's row of the table; zeros where nothing is rotated.
template <int VEC, bool INTER>
__device__ __forceinline__ void load_angles(const float *row, int u, int oa, int ob, Turned t, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = t.lo ? row[u] : 0.0f;
    } else {
        constexpr int H = VEC / 2;
        float lo[H] = {}, hi[H] = {};
        if (t.lo) load_floats<H>(row + (INTER ? oa / 2 : u * VEC), lo);
        if (t.hi) load_floats<H>(row + (INTER ? ob / 2 : u * VEC + H), hi);
#pragma unroll
        for (int j = 0; j < H; ++j) {
            v[j] = lo[j];
            v[H + j] = hi[j];
        }
    }
}

// (x, y) -> (x' k0 - y' k1, y' k2 + x' k3), x' = scale x, y' = scale y: norm, weights and rotation
// of a pair in one step, with k0 = w_x cos, k1 = w_y sin, k2 = w_y cos, k3 = w_x sin.  The scale goes
// first: normed items are at most sqrt(dim), so that no product here leaves float32's range where
// the result does not, and the zero scale of a head whose squares did gives zeros.  Pairs that are
// not rotated take their weights k0, k2 alone: a product with a zero sine would carry an infinity
// over to the partner.
template <int FROM, int TO, int VEC>
__device__ __forceinline__ void turn(float (&x)[VEC], float (&y)[VEC], const float (&k0)[VEC], const float (&k1)[VEC],
                                     const float (&k2)[VEC], const float (&k3)[VEC], float scale, bool turned) {
    if constexpr (TO - FROM == 1) {
        x[FROM] *= scale;
        y[FROM] *= scale;
        const float u = turned ? x[FROM] * k0[FROM] - y[FROM] * k1[FROM] : x[FROM] * k0[FROM];
        const float v = turned ? y[FROM] * k2[FROM] + x[FROM] * k3[FROM] : y[FROM] * k2[FROM];
        x[FROM] = u;
        y[FROM] = v;
    } else {
        const float2 by = make_float2(scale, scale);
#pragma unroll
        for (int j = FROM; j < TO; j += 2) {
            const float2 xx = mul2(make_float2(x[j], x[j + 1]), by), yy = mul2(make_float2(y[j], y[j + 1]), by);
            float2 u = mul2(xx, make_float2(k0[j], k0[j + 1])), v = mul2(yy, make_float2(k2[j], k2[j + 1]));
            if (turned) {
                u = fma2(make_float2(-yy.x, -yy.y), make_float2(k1[j], k1[j + 1]), u);
                v = fma2(xx, make_float2(k3[j], k3[j + 1]), v);
            }
            x[j] = u.x;
            x[j + 1] = u.y;
            y[j] = v.x;
            y[j + 1] = v.y;
        }
    }
}

// sum of the squares of a and b, on top of `sum`
template <int VEC>
__device__ __forceinline__ float squares(const float (&a)[VEC], const float (&b)[VEC], float sum) {
    if constexpr (VEC == 1) {
        return sum + (a[0] * a[0] + b[0] * b[0]);
    } else {
        float2 s = make_float2(sum, 0.0f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 x = make_float2(a[j], a[j + 1]), y = make_float2(b[j], b[j + 1]);
            s = fma2(x, x, s);
            s = fma2(y, y, s);
        }
        return s.x + s.y;
    }
}

// ---- quantisation -----------------------------------------------------------------
__device__ __forceinline__ uint32_t pack_codes2(float hi, float lo, int e5m2) {
    uint16_t r;
    if (e5m2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&v)[VEC], float by, int e5m2) {
    if constexpr (VEC == 1) {
        *p = static_cast<uint8_t>(pack_codes2(0.0f, v[0] * by, e5m2));
    } else {
        Chunk<uint8_t, VEC> c;
        const float2 by2 = make_float2(by, by);
        if constexpr (VEC == 2) {
            const float2 x = mul2(make_float2(v[0], v[1]), by2);
            c.all = static_cast<uint16_t>(pack_codes2(x.y, x.x, e5m2));
        } else {
#pragma unroll
            for (int j = 0; j < VEC / 4; ++j) {
                const float2 x = mul2(make_float2(v[4 * j], v[4 * j + 1]), by2);
                const float2 y = mul2(make_float2(v[4 * j + 2], v[4 * j + 3]), by2);
                c.word[j] = pack_codes2(x.y, x.x, e5m2) | (pack_codes2(y.y, y.x, e5m2) << 16);
            }
        }
        *reinterpret_cast<typename Chunk<uint8_t, VEC>::Word *>(p) = c.all;
    }
}

// Largest magnitude of a and of m; NaNs do not count, infinities do.  sm_100 takes the
// maximum of three magnitudes in one instruction.
template <int VEC>
__device__ __forceinline__ float largest(const float (&a)[VEC], float m) {
    if constexpr (VEC == 1) {
        m = fmaxf(m, fabsf(a[0]));
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a[j]), "f"(a[j + 1]));
    }
    return m;
}
// The same without infinities: an infinity says nothing about the scale.
template <int VEC>
__device__ __forceinline__ float largest_finite(const float (&a)[VEC], float m) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float x = fabsf(a[j]);
        m = fmaxf(m, x <= FLT_MAX ? x : 0.0f);
    }
    return m;
}

// The scale of a largest magnitude, and its reciprocal.  The lower bound 2^-126 keeps the
// reciprocal finite and covers a row of zeros.
struct Scale {
    float value, inverse;
    __device__ Scale(float amax, int e5m2, int e8m0) {
        if (e8m0) {
            // amax / largest rounded up to a power of two.  largest = 1.75 * 2^8 or
            // 1.75 * 2^15, so the quotient's power is that of amax, less 8 or 15, one more
            // if amax's mantissa is above 1.75; the rounding of the quotient to float32
            // cannot change this, since the float32 after 1.75 * 2^k is 1.75 * 2^k *
            // (1 + 0.57 * 2^-23).  A field of at most 247 leaves a normal reciprocal.
            const int field = static_cast<int>((__float_as_uint(amax) + 0x001FFFFFu) >> 23) - (e5m2 ? 15 : 8);
            const uint32_t e = static_cast<uint32_t>(max(field, 1));
            value = __uint_as_float(e << 23);
            inverse = __uint_as_float((254u - e) << 23);
        } else {
            value = fmaxf(__fdiv_rn(amax, e5m2 ? 57344.0f : 448.0f), 0x1p-126f);
            inverse = __frcp_rn(value);
        }
    }
    __device__ void store(void *scales, int64_t at, int e8m0) const {
        if (e8m0) static_cast<uint8_t *>(scales)[at] = static_cast<uint8_t>(__float_as_uint(value) >> 23);
        else static_cast<float *>(scales)[at] = value;
    }
};

// ---- host side ----------------------------------------------------------------------
// The (items per chunk, units per lane) pairs that are compiled; choose() picks one.
// Chunks of 8 are for 16-bit items only (16 bytes).
#define B2K_HEADS_SHAPES(CASE) \
    CASE(8, 1) CASE(8, 2) CASE(4, 1) CASE(4, 4) CASE(2, 1) CASE(2, 4) CASE(1, 1) CASE(1, 4) CASE(1, 16)

struct Plan {
    int vec = 0, iter = 0;
};

// Argument checks; the messages start with `name`.  0 = fine.
int item_bytes(int64_t format);                      // 0 for a format that arrays of heads cannot have
int check_heads(const b2k_heads &h, const char *name, const char *what, int64_t tokens, int itemsize, bool written);
int check_like(const b2k_heads &h, const b2k_heads &like, const char *name, const char *what);
// Two outputs that start at one address would overwrite each other.
int check_apart(const void *a, const void *b, const char *name, const char *what);
int check_tokens(int64_t format, int64_t tokens, const char *name);
int check_rotation(const b2k_rotation *r, const char *name);
int check_cache(const b2k_cache *c, const char *name);
int check_side(const b2k_pages &side, const b2k_heads &like, const b2k_cache &c, const char *name, const char *what,
               bool written);
int check_indices(const void *p, int64_t bytes, const char *name, const char *what);

void set_input(Role &r, const b2k_heads &h, int64_t tokens);
void set_output(Role &r, const b2k_heads &h, int64_t tokens);
void set_grad(Role &r, const b2k_heads &h, int64_t tokens);
void set_pages(Params &p, Role &r, const b2k_cache &c, const b2k_pages &side);
void set_rotation(Params &p, const b2k_rotation &rot);
// Widest chunks that a role's sizes, strides and addresses allow.
int widest(const Params &p, int which, int64_t format, const b2k_rotation *rot);
// Lanes and unit layout of every role for chunks of `vec` items, or fewer.
Plan lay_out(Params &p, int vec, const b2k_rotation *rot);
// Items with up to `most` heads in each, fewer where `busy` threads an SM would not have
// work, and blocks of every role; an error when they do not fit 31 bits.
int count_items(Params &p, int most, int busy, const char *name);

}  // namespace headwise
