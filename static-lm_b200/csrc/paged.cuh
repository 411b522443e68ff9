// paged.cuh -- the paged key/value cache as the kernels see it: pages of
// [kv_head][slot][head_dim], a table of page ids per sequence, and rows of
// activations laid end to end over the sequences.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace slm {

// KV_Q8: signed bytes, then an f32 scale per (KV head, slot) at scale_at; an
// element of its strides and offsets is a byte.
enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2, KV_Q8 = 3 };
// bits of the status word
constexpr int PAGED_BAD_PAGE = 1;      // a page id at or past num_pages, or none where one is written
constexpr int PAGED_BAD_POSITION = 2;  // a position past the page table or the rope table
constexpr int PAGED_WAIT_GAVE_UP = 4;  // a bounded device wait gave up
constexpr int PAGED_BAD_ROWS = 8;      // row_start is negative, falls, or ends past num_rows

constexpr float NO_MAX = -FLT_MAX;  // a running maximum before any key: no finite score is below it

struct KvView {
    void *k, *v;
    uint64_t page_stride;  // elements
    int num_pages, page_size;
    int page_shift;  // log2(page_size), or -1
    int kv_heads, hd, type;
    int32_t *status;
    uint64_t scale_at;  // KV_Q8: byte offset of a page's scales
};

struct BatchView {
    const int32_t *row_start;  // null: row i is sequence i's one new row
    const int32_t *kv_len, *table;
    unsigned table_stride;
    int num_seqs, num_rows;
    int cap;  // positions a row of the page table covers
};

__device__ __forceinline__ void paged_flag(const KvView &kv, int bit) {
    if (kv.status) atomicOr(kv.status, bit);
}

// Sequence and position of an activation row; position -1 for a row that
// belongs to no sequence or lies before its sequence's start.  (A sequence
// whose rows end past num_rows keeps their positions.)
__device__ __forceinline__ void row_place(const KvView &kv, const BatchView &b, int row, int &seq, int &pos) {
    seq = row;
    if (!b.row_start) {
        pos = b.kv_len[row] - 1;
        return;
    }
    int lo = 0, hi = b.num_seqs;  // the last s with row_start[s] <= row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.row_start[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    seq = lo;
    const int end = b.row_start[lo + 1];
    if (end > b.num_rows) paged_flag(kv, PAGED_BAD_ROWS);
    pos = b.row_start[lo] <= row && row < end ? b.kv_len[lo] - (end - row) : -1;
}

__device__ __forceinline__ unsigned page_index(const KvView &kv, unsigned key) {
    return kv.page_shift >= 0 ? key >> kv.page_shift : key / (unsigned)kv.page_size;
}

// The page of (sequence, key) and the key's slot in it, or -1 where the key's
// page is not held (a negative id) or the id or the key is out of range (the
// latter two set the status word).
__device__ __forceinline__ int key_page(const KvView &kv, const BatchView &b, int seq, unsigned key, unsigned &slot) {
    const unsigned pi = page_index(kv, key);
    slot = key - pi * (unsigned)kv.page_size;
    if (pi >= b.table_stride) {
        paged_flag(kv, PAGED_BAD_POSITION);
        return -1;
    }
    const int page = b.table[(size_t)seq * b.table_stride + pi];
    if ((unsigned)page >= (unsigned)kv.num_pages) {
        if (page >= 0) paged_flag(kv, PAGED_BAD_PAGE);
        return -1;
    }
    return page;
}
__device__ __forceinline__ long long row_offset(const KvView &kv, int page, int head, unsigned slot) {
    return (long long)((uint64_t)page * kv.page_stride +
                       ((uint64_t)head * (unsigned)kv.page_size + slot) * (unsigned)kv.hd);
}
// A load that is issued here, not where its result is used.
__device__ __forceinline__ unsigned ldg_now(const void *p) {
    unsigned v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Byte offset of the row's scale (KV_Q8).
__device__ __forceinline__ long long scale_offset(const KvView &kv, int page, int head, unsigned slot) {
    return (long long)((uint64_t)page * kv.page_stride + kv.scale_at +
                       ((uint64_t)head * (unsigned)kv.page_size + slot) * 4u);
}
__device__ __forceinline__ float scale_get(const void *pool, long long at) {
    return *reinterpret_cast<const float *>(reinterpret_cast<const char *>(pool) + at);
}
// Element offset of (sequence, key, KV head) in the pools, or -1 as key_page.
__device__ __forceinline__ long long key_offset(const KvView &kv, const BatchView &b, int seq, unsigned key, int head) {
    unsigned slot;
    const int page = key_page(kv, b, seq, key, slot);
    return page < 0 ? -1 : row_offset(kv, page, head, slot);
}

// The keys that rows at positions first_pos..last_pos (the first may be
// negative) see between them, as a list of n: the sinks, then from the first
// row's window on (window 0: from the start) up to the last row.  Positions
// past the page table are none.
struct SeenKeys {
    int sinks, low, n;  // list index i -> i < sinks ? i : i - sinks + low
    __device__ __forceinline__ int key(int i) const { return i < sinks ? i : i - sinks + low; }
};
__device__ __forceinline__ SeenKeys seen_keys(const BatchView &b, int first_pos, int last_pos, unsigned window, unsigned sinks) {
    SeenKeys s;
    const int end = last_pos < b.cap ? last_pos + 1 : b.cap;
    s.low = 0;
    if (window != 0 && first_pos >= 0 && (unsigned)first_pos >= window) s.low = first_pos - (int)window + 1;
    if (end > 0 && s.low > end) s.low = end;
    s.sinks = (unsigned)s.low < sinks ? s.low : (int)sinks;
    s.n = end > 0 ? s.sinks + end - s.low : 0;
    return s;
}

// ---- packed f32 pairs: two roundings in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// ---- f32 values as sums of 16-bit parts
// bf16: every part is what the ones before it leave; the exponents are f32's.
// f16: the first part and 2^12 times what it leaves.  f16 ends at 2^-24, so
// that an unscaled second part of a value below 2^-2 would keep fewer and fewer
// bits and none of one below 2^-25; scaled, the parts hold values from 2^-14
// (where the first one's own bits begin to go) to 2^15 to 2^-24 of themselves
// and smaller ones to 2^-37.
constexpr float F16_PART2 = 4096.0f, F16_PART2_INV = 1.0f / 4096.0f;
constexpr int F16_PART2_LOG2 = 12;
// Where a softmax's weights 2^(x - m) lie: m is set `margin` below the largest
// score, and set anew once a score passes it by `rescale`.  bf16 parts and f32
// weights have room on either side.  f16 parts need the weights as high as
// their type goes: at most 2^15, a row's largest at least 2^9, so that weights
// down to 2^-23 of it are held to 2^-24 of themselves and smaller ones to 2^-46
// of it: those of e^-17 beside one of 1 to 3e-7 of themselves, those of e^-20 to
// 7e-6.  (At most 2^8, the largest at least 1, with an unscaled second part: 40 %
// and nothing left.)  Each bit less between margin and rescale doubles that
// range and has references move more often: 8 x 4096 rows of 9 / 3 heads of 64
// 644 us with 7, 645 with 6, 653 with 5, 678 with 4.
template <int TYPE>
struct WeightRange {
    static constexpr float margin = TYPE == KV_F16 ? 9.0f : 0.0f, rescale = TYPE == KV_F16 ? 15.0f : 8.0f;
    static constexpr float least = TYPE == KV_F16 ? 256.0f : 0.5f;  // half of 2^margin
};

// Two f32 values as the packed 16-bit parts of an operand.  (The second part
// of an infinity is NaN: rows that meet it come out NaN and are redone.)
template <int TYPE, int N>
__device__ __forceinline__ void split2(float a, float b, unsigned (&part)[N]) {
    if constexpr (TYPE == KV_F16) {
        static_assert(N == 2, "two parts");
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        float ra, rb;  // (a - f) 2^12, exact
        unpack2(fma2(pack2(f.x, f.y), pack2(-F16_PART2, -F16_PART2), mul2(pack2(a, b), pack2(F16_PART2, F16_PART2))), ra, rb);
        const __half2 r = __floats2half2_rn(ra, rb);
        part[0] = *reinterpret_cast<const unsigned *>(&h);
        part[1] = *reinterpret_cast<const unsigned *>(&r);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            part[i] = *reinterpret_cast<const unsigned *>(&h);
            if (i + 1 < N) {
                a = __fsub_rn(a, __uint_as_float(part[i] << 16));
                b = __fsub_rn(b, __uint_as_float(part[i] & 0xffff0000u));
            }
        }
    }
}
// The same of f16, what the first part leaves by multiply-adds that take it as it is
// (two instructions fewer): b's in the upper halves.
__device__ __forceinline__ void split2_f16(float a, float b, unsigned &first, unsigned &second) {
    const __half2 h = __floats2half2_rn(a, b);
    first = *reinterpret_cast<const unsigned *>(&h);
    float ra, rb;
    unpack2(mul2(pack2(a, b), pack2(F16_PART2, F16_PART2)), ra, rb);
    asm("{\n .reg .b16 x, y, c;\n mov.b32 {x, y}, %2;\n mov.b16 c, 0xEC00;\n"  // -4096
        " fma.rn.f32.f16 %0, x, c, %0;\n fma.rn.f32.f16 %1, y, c, %1;\n}\n"
        : "+f"(ra), "+f"(rb)
        : "r"(first));
    const __half2 r = __floats2half2_rn(ra, rb);
    second = *reinterpret_cast<const unsigned *>(&r);
}
static_assert(F16_PART2 == 4096.0f, "the constant above");

// The same of two softmax weights (finite, or NaN: then the row is redone).
template <int TYPE, int N>
__device__ __forceinline__ void split2_weights(float a, float b, unsigned (&part)[N]) {
    if constexpr (TYPE == KV_F16) {
        split2<KV_F16, N>(a, b, part);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {  // cut, not rounded: 8 bits each
            const unsigned ua = __float_as_uint(a), ub = __float_as_uint(b);
            part[i] = __byte_perm(ua, ub, 0x7632);
            if (i + 1 < N) {
                a = __fsub_rn(a, __uint_as_float(ua & 0xffff0000u));
                b = __fsub_rn(b, __uint_as_float(ub & 0xffff0000u));
            }
        }
    }
}

// Four values to / from a page's element type.
template <int TYPE>
struct KvElem;
template <>
struct KvElem<KV_F32> {
    using T = float;
    static __device__ __forceinline__ void store4(float *p, const float (&x)[4]) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
};
template <>
struct KvElem<KV_F16> {
    using T = __half;
    // rounded to nearest even, past the largest f16 to infinity: the type's own conversion
    static __device__ __forceinline__ void store4(__half *p, const float (&x)[4]) {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
    static __device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
};
template <>
struct KvElem<KV_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&x)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
    static __device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};
template <>
struct KvElem<KV_Q8> {
    using T = int8_t;
    static __device__ __forceinline__ float get(const int8_t *p) { return (float)*p; }
};

// The 8-bit kernels sum bytes times q 2^e, whose largest element is below 2^15, and
// take 2^-e back after the key's scale: |sum| < 2^15 127 128 < 2^29, so that the
// product with a scale below 2^98 is finite, while with a larger one it may pass f32
// where the score itself does not.  Rows that see such a key are redone.
constexpr unsigned Q8_KEY_LIMIT = (unsigned)(127 + 98) << 23;
__device__ __forceinline__ unsigned q8_above_limit(float scale) { return __float_as_uint(fabsf(scale)) - Q8_KEY_LIMIT; }
__device__ __forceinline__ bool q8_large_key(unsigned above_limit) { return above_limit < 0x7f800000u - Q8_KEY_LIMIT; }

// Their weights, times a value's scale relative to a power of two at or above its
// tile's largest, are two f16 parts, off by up to 2^-37, and times bytes by 2^-30 a key.
// Scales beside them that a row does not see, or sees with next to no weight, so take
// bits of its own; a row whose sums of n keys all come out below 2^-5 of the largest
// power of two (where a row's largest weight is 2^9 or more: its result is below 2^-21
// of the largest value) is redone.  What is left is off by n 2^-25 at most, sqrt(n) 2^-27
// as a rule.
constexpr float Q8_RESULT_LEAST = 1.0f / 32;

// One row and query head over the keys [lo, hi) of a list, of which it sees
// those below sink_end and those in [from, to), on the CUDA cores by one warp:
// 32 keys at a time, a key per lane for the scores, head_dim over the lanes
// for the values.  The tensor-core kernels redo so what came out not finite:
// 0 x NaN of a key in the tile that a row does not see reaches it there, and
// the parts of an infinity are not its parts.  (Scores of 8-bit keys in 64 bits
// until their last factor: neither the sum nor the scale is near their ends.)
struct RowState {
    float m, l, acc[4];
};
template <int TYPE>
__device__ __noinline__ RowState attend_row(const KvView &kv, const BatchView &b, int seq, int head, const float *q,
                                            float sl2, SeenKeys keys, int lo, int hi, int from, int sink_end, int to) {
    using T = typename KvElem<TYPE>::T;
    const int lane = threadIdx.x & 31, hd = kv.hd;
    RowState r;
    r.m = NO_MAX;
    r.l = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) r.acc[c] = 0.f;
    if (hi > to) hi = to;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        long long off = -1;
        float v_scale = 1.0f;
        float x = -INFINITY;
        if (i < hi && (i < sink_end || i >= from)) {
            unsigned slot;
            const int page = key_page(kv, b, seq, (unsigned)keys.key(i), slot);
            if (page >= 0) {
                off = row_offset(kv, page, head, slot);
                const T *k = reinterpret_cast<const T *>(kv.k) + off;
                if constexpr (TYPE == KV_Q8) {
                    double dot = 0.0;
                    for (int d = 0; d < hd; d++) dot = fma((double)q[d], (double)KvElem<TYPE>::get(k + d), dot);
                    const long long at = scale_offset(kv, page, head, slot);
                    x = (float)(dot * (double)scale_get(kv.k, at) * (double)sl2);
                    v_scale = scale_get(kv.v, at);
                } else {
                    float dot = 0.f;
                    for (int d = 0; d < hd; d++) dot = __fmaf_rn(q[d], KvElem<TYPE>::get(k + d), dot);
                    x = __fmul_rn(dot, sl2);
                }
            }
        }
        float top = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, r.m);
        const float f = exp2_approx(__fsub_rn(r.m, top)), w = exp2_approx(__fsub_rn(x, top));
        r.m = top;
        float total = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total = __fadd_rn(total, __shfl_xor_sync(0xffffffffu, total, o));
        r.l = __fmaf_rn(r.l, f, total);
#pragma unroll
        for (int c = 0; c < 4; c++) r.acc[c] = __fmul_rn(r.acc[c], f);
        const float wv = TYPE == KV_Q8 ? __fmul_rn(w, v_scale) : w;
        for (int j = 0; j < 32; j++) {
            const long long o = __shfl_sync(0xffffffffu, off, j);
            const float wj = __shfl_sync(0xffffffffu, wv, j);
            if (o < 0) continue;
            const T *v = reinterpret_cast<const T *>(kv.v) + o;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (lane + 32 * c < hd) r.acc[c] = __fmaf_rn(wj, KvElem<TYPE>::get(v + lane + 32 * c), r.acc[c]);
        }
    }
    return r;
}

}  // namespace slm
