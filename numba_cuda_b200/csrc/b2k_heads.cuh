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

constexpr int kThreads = 256;

// Rows of one token that a group keeps in flight: cosines, sines and weights are loaded
// once for all of them.  Rows that spread over several units a lane leave registers for
// fewer.
B2K_HD constexpr int rows_in_flight(int iter) { return iter == 1 ? 4 : iter == 2 ? 2 : 1; }

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
    int angle_units;            // units below it are rotated
    int scale_lanes, scale_joint;     // lanes that share a scale (0: found through shared memory), and whether
                                      // a lane's two chunks do
    float inv_dim;
};

struct Params {
    Role role[3];
    int64_t tokens;
    int heads_per_item, lanes, lane_bits;
    int norm, interleaved, weight_format;
    float eps;
    const float *cos_table, *sin_table;
    int64_t cos_stride, sin_stride, table_rows;
    const void *positions;
    int position_bytes;
    const void *slots;
    int slot_bytes, e5m2, e8m0;
    int64_t pages, page_size;
    float *partials;            // backward: weight-gradient partial sums, one row of dim floats per block
    int blocks0;                // backward: blocks of role 0
};

template <typename T> struct Convert;
template <> struct Convert<float> {
    __device__ static float up(float x) { return x; }
    __device__ static float down(float x) { return x; }
};
template <> struct Convert<__half> {
    __device__ static float up(__half x) { return __half2float(x); }
    __device__ static __half down(float x) { return __float2half_rn(x); }
    using Pair = __half2;
    __device__ static __half2 down2(float lo, float hi) { return __floats2half2_rn(lo, hi); }
};
template <> struct Convert<__nv_bfloat16> {
    // a bfloat16 is the upper half of a float32: a shift.  The conversion instruction runs on
    // the quarter-rate unit that divisions and square roots use and was what bounded the
    // first kernels (unit busy 100%, DRAM 28%).
    __device__ static float up(__nv_bfloat16 x) {
        return __uint_as_float(static_cast<uint32_t>(__bfloat16_as_ushort(x)) << 16);
    }
    __device__ static __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
    using Pair = __nv_bfloat162;
    __device__ static __nv_bfloat162 down2(float lo, float hi) { return __floats2bfloat162_rn(lo, hi); }
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
    T e[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T *p) {
    return *reinterpret_cast<const Chunk<T, VEC> *>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T *p, const float (&v)[VEC]) {
    Chunk<T, VEC> c;
    if constexpr (VEC > 1 && sizeof(T) == 2) {        // two items per conversion instruction
        Chunk<typename Convert<T>::Pair, VEC / 2> two;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) two.e[j] = Convert<T>::down2(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<Chunk<typename Convert<T>::Pair, VEC / 2> *>(p) = two;
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) c.e[j] = Convert<T>::down(v[j]);
        *reinterpret_cast<Chunk<T, VEC> *>(p) = c;
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Chunk<T, VEC> &c, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = Convert<T>::up(c.e[j]);
}

template <int VEC>
__device__ __forceinline__ void load_floats(const float *p, float (&v)[VEC]) {
    constexpr int W = VEC < 4 ? VEC : 4;       // 16 bytes at most
#pragma unroll
    for (int j = 0; j < VEC; j += W) {
        const Chunk<float, W> c = load_chunk<float, W>(p + j);
#pragma unroll
        for (int i = 0; i < W; ++i) v[j + i] = c.e[i];
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

// The lanes of a group, and where a unit's two chunks start.
struct Lanes {
    int n, lane;
    unsigned mask;
    __device__ explicit Lanes(int lanes) : n(lanes), lane(threadIdx.x & (lanes - 1)) {
        const unsigned ones = lanes == 32 ? 0xFFFFFFFFu : (1u << lanes) - 1u;
        mask = ones << ((threadIdx.x & 31) & ~(lanes - 1));
    }
    __device__ float sum(float v) const {
        for (int o = n >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
        return v;
    }
    // over aligned runs of `span` lanes (a power of two) of the group
    __device__ float max(float v, int span) const {
        for (int o = span >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
        return v;
    }
};

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

// Rotation of a unit by its angles (VEC == 1: a pair is always the unit's two items).
template <int VEC>
__device__ __forceinline__ void rotate(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC],
                                       bool interleaved) {
    if (VEC == 1 || !interleaved) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float x = a[j], y = b[j];
            a[j] = x * c[j] - y * s[j];
            b[j] = y * c[j] + x * s[j];
        }
    } else if constexpr (VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            float x = a[2 * j], y = a[2 * j + 1];
            a[2 * j] = x * c[j] - y * s[j];
            a[2 * j + 1] = y * c[j] + x * s[j];
            x = b[2 * j], y = b[2 * j + 1];
            b[2 * j] = x * c[VEC / 2 + j] - y * s[VEC / 2 + j];
            b[2 * j + 1] = y * c[VEC / 2 + j] + x * s[VEC / 2 + j];
        }
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
        Chunk<uint16_t, VEC / 2> c;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) c.e[j] = pack_codes2(v[2 * j + 1] * by, v[2 * j] * by, e5m2);
        *reinterpret_cast<Chunk<uint16_t, VEC / 2> *>(p) = c;
    }
}

template <int VEC>
__device__ __forceinline__ float largest_finite(const float (&v)[VEC]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float x = fabsf(v[j]);
        m = fmaxf(m, x <= FLT_MAX ? x : 0.0f);      // an infinity or a NaN says nothing about the scale
    }
    return m;
}

// The scale of a largest magnitude, and its reciprocal.  The lower bound keeps the
// reciprocal finite and covers a row of zeros.
struct Scale {
    float value, inverse;
    __device__ Scale(float amax, int e5m2, int e8m0) {
        value = fmaxf(__fdiv_rn(amax, e5m2 ? 57344.0f : 448.0f), 0x1p-126f);
        if (e8m0) {
            // a normal number: adding all mantissa bits carries into the exponent unless
            // they are all zero, which is the power of two not below it.  Its exponent
            // field is at most 127 + 120, so the reciprocal is a normal number, too.
            const uint32_t e = (__float_as_uint(value) + 0x007FFFFFu) >> 23;
            value = __uint_as_float(e << 23);
            inverse = __uint_as_float((254u - e) << 23);
        } else {
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
#define B2K_HEADS_SHAPES(CASE) CASE(8, 1) CASE(8, 2) CASE(4, 1) CASE(4, 4) CASE(1, 1) CASE(1, 4) CASE(1, 16)

struct Plan {
    int vec = 0, iter = 0;
};

// Argument checks; the messages start with `name`.  0 = fine.
int item_bytes(int64_t format);                      // 0 for a format that arrays of heads cannot have
int check_heads(const b2k_heads &h, const char *name, const char *what, int64_t tokens, int itemsize, bool written);
int check_like(const b2k_heads &h, const b2k_heads &like, const char *name, const char *what);
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
// Chunk width from sizes, strides and addresses; lanes and unit layout of every role.
Plan choose(Params &p, int64_t format, const b2k_rotation *rot);
// Items with up to `most` heads in each, and blocks of `threads` threads, of every role; an
// error when they do not fit 31 bits.
int count_items(Params &p, int most, int threads, const char *name);

}  // namespace headwise
