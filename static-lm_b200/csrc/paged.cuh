// paged.cuh -- the paged key/value cache as the kernels see it: pages of
// [kv_head][slot][head_dim], a table of page ids per sequence, and rows of
// activations laid end to end over the sequences.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace slm {

enum KvType : int { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };
// bits of the status word
constexpr int PAGED_BAD_PAGE = 1;      // a page id at or past num_pages, or none where one is written
constexpr int PAGED_BAD_POSITION = 2;  // a position past the page table or the rope table
constexpr int PAGED_WAIT_GAVE_UP = 4;  // a bounded device wait gave up

struct KvView {
    void *k, *v;
    uint64_t page_stride;  // elements
    int num_pages, page_size;
    int page_shift;  // log2(page_size), or -1
    int kv_heads, hd, type;
    int32_t *status;
};

struct BatchView {
    const int32_t *row_start;  // null: row i is sequence i's one new row
    const int32_t *kv_len, *table;
    unsigned table_stride;
    int num_seqs, num_rows;
};

__device__ __forceinline__ void paged_flag(const KvView &kv, int bit) {
    if (kv.status) atomicOr(kv.status, bit);
}

// Sequence and position of an activation row; position -1 for a row that
// belongs to no sequence or lies before its sequence's start.
__device__ __forceinline__ void row_place(const BatchView &b, int row, int &seq, int &pos) {
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
    pos = b.row_start[lo] <= row && row < end ? b.kv_len[lo] - (end - row) : -1;
}

__device__ __forceinline__ unsigned page_index(const KvView &kv, unsigned key) {
    return kv.page_shift >= 0 ? key >> kv.page_shift : key / (unsigned)kv.page_size;
}

// Element offset of (sequence, key, KV head) in the pools, or -1 where the
// key's page is not held (a negative id) or the id or the key is out of
// range (the latter two set the status word).
__device__ __forceinline__ long long key_offset(const KvView &kv, const BatchView &b, int seq, unsigned key, int head) {
    const unsigned pi = page_index(kv, key);
    if (pi >= b.table_stride) {
        paged_flag(kv, PAGED_BAD_POSITION);
        return -1;
    }
    const int page = b.table[(size_t)seq * b.table_stride + pi];
    if ((unsigned)page >= (unsigned)kv.num_pages) {
        if (page >= 0) paged_flag(kv, PAGED_BAD_PAGE);
        return -1;
    }
    const unsigned slot = key - pi * (unsigned)kv.page_size;
    return (long long)((uint64_t)page * kv.page_stride +
                       ((uint64_t)head * (unsigned)kv.page_size + slot) * (unsigned)kv.hd);
}

// The keys a row at position p sees, as a list of n_seen: key j of the list
// is j below the sink count, and counts on from the window's first key after
// it.  window 0 = every key up to p.
struct SeenKeys {
    int sinks, low, n;  // list index i -> i < sinks ? i : i - sinks + low
    __device__ __forceinline__ int key(int i) const { return i < sinks ? i : i - sinks + low; }
};
__device__ __forceinline__ SeenKeys seen_keys(int first_pos, int last_pos, unsigned window, unsigned sinks) {
    // union over rows at first_pos..last_pos (first_pos may be negative)
    SeenKeys s;
    const int end = last_pos + 1;
    s.low = 0;
    if (window != 0 && first_pos >= 0 && (unsigned)first_pos >= window) s.low = first_pos - (int)window + 1;
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

}  // namespace slm
