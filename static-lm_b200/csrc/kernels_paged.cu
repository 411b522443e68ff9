// kernels_paged.cu -- the paged key/value cache: new keys and values into
// their pages with the per-head RMSNorm and the position rotation applied on
// the way.
#include "async.cuh"
#include "kernels.h"

namespace slm {

namespace {

constexpr int AP_THREADS = 256;

__device__ __forceinline__ void load4(const float *p, bool vec, float (&x)[4]) {
    if (vec) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = p[j];
    }
}

__device__ __forceinline__ void turn(float &p, float &q, float c, float s) {
    const float t = __fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s));
    q = __fadd_rn(__fmul_rn(p, s), __fmul_rn(q, c));
    p = t;
}

// LPV lanes (a power of two, 8 elements each) per head vector; the vectors of
// a row are its query heads, its key heads, then its value heads.
//   norm:  y = x * (1 / sqrt(sum(x^2) / head_dim + eps)) * w      (q and k)
//   turn:  (a, b) -> (a cos - b sin, a sin + b cos)                (q and k)
// with (a, b) neighbours, or the two halves of the first rotary_dim elements.
// Every product and sum is rounded on its own, so that the rotation gives the
// bits of slm_apply_rope_cached.
//
// A group of LPV lanes takes AP_VECS vectors of one row: what they share (the
// row's place, found by a search in row_start, its page's offset, its row of
// the rope tables) is worked out once for them, with all their loads in flight.
// 8 bytes in and out per query element, 4 + the page's type per key and value
// element are its bytes.  With a vector a group it was bound by instructions
// (issue 77 % of the cycles, DRAM 49 %; now 62 and 56).  With one, two, three and
// four vectors a group (64 registers each), prompts of 4096 rows into f16
// pages:
//   8 x 9 + 3 + 3 heads of 64          49.9  44.5  43.1  44.8 us (f32 pages 45.4, bf16 43.1)
//   2 x 32 + 8 + 8 of 128, normed      83.8  75.0  73.7  73.5
//   8 x 6 + 6 + 6 of 48                57.3  49.0  43.1  46.9 (two of eight lanes idle)
//   6 x 12 + 2 + 2 of 80               69.6  56.7  52.4  49.9 (six of sixteen)
//   4 x 20 + 4 + 4 of 96               81.8  67.8  63.8  61.5 (four of sixteen)
//   12 x 4 + 4 + 4 of 32, bf16 pages   34.8  30.6  28.2  28.7
// Three are best or within 5 % everywhere: 4.5 to 5.7 TB/s.  Single rows are one
// launch's time.  8-bit pages (amax and two quotients a vector on top: issue, not
// memory, bounds them): one, two, three 61.8, 48.0, 50.0 us for the first (without
// the quotients 46.8).
template <int TYPE>
constexpr int AP_VECS = TYPE == KV_Q8 ? 2 : 3;

// 8-bit rows: x = q scale with scale = max|x| / 127 and q = x (127 / max|x|)
// rounded to the nearest, ties to even: off by half a step, max|x| / 254, and
// the roundings of the two quotients and the product.  A row of magnitudes
// below 2^-100, whose scale would be near f32's smallest, is stored as zeros; one
// that holds an infinity or a NaN as NaN throughout, by its scale.
struct Q8Row {
    float scale, up;
};
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ Q8Row q8_row(unsigned top) {
    Q8Row r;
    r.scale = r.up = 0.f;
    if (top >= 0x7f800000u) {
        r.scale = __uint_as_float(0x7fc00000u);
    } else if (top >= (unsigned)(127 - 100) << 23) {
        // max|x| / 127 rounded once: the quotient by the rounded 1/127 and what its exact
        // remainder adds (Markstein's theorem); a third of the division's instructions
        const float a = __uint_as_float(top), y = 1.0f / 127.0f, q = __fmul_rn(a, y);
        r.scale = __fmaf_rn(__fmaf_rn(-127.0f, q, a), y, q);
        r.up = __fdiv_rn(127.0f, __uint_as_float(top));
    }
    return r;
}
__device__ __forceinline__ unsigned q8_pack(const float (&x)[4], float up) {
    // 1.5 2^23 + q: q is rounded to the nearest by the sum, and its low byte is the sum's
    unsigned u[4];
#pragma unroll
    for (int j = 0; j < 4; j++) u[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[j], up), 12582912.0f));
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
}

template <int TYPE, int LPV>
__global__ void __launch_bounds__(AP_THREADS, 4) paged_append_kernel(KvView kv, BatchView b, AppendView a) {
    using T = typename KvElem<TYPE>::T;
    if constexpr (TYPE == KV_Q8) {
        pdl_wait();
        pdl_release();
    }
    const int l = threadIdx.x % LPV, hd = kv.hd;
    const int per_row = a.num_heads + 2 * kv.kv_heads, parts = (per_row + AP_VECS<TYPE> - 1) / AP_VECS<TYPE>;
    const unsigned item = blockIdx.x * (AP_THREADS / LPV) + threadIdx.x / LPV;  // below 2^32: the host's check
    const unsigned its_row = item / (unsigned)parts;
    const bool live = its_row < (unsigned)b.num_rows && l * 8 < hd;
    const int row = live ? (int)its_row : 0;
    const int first = live ? (int)(item - its_row * (unsigned)parts) * AP_VECS<TYPE> : 0;
    const int rd = a.rotary_dim;
    const bool turns = 8 * l < rd;          // this lane's elements of q and k are rotated,
    const bool split = turns && a.halves;   // as pairs half of rotary_dim apart
    const int i0 = split ? 4 * l : 8 * l, i1 = split ? rd / 2 + 4 * l : 8 * l + 4;
    const float *const rq = a.q + (size_t)row * a.ldq, *const rk = a.k + (size_t)row * a.ldk,
                *const rv = a.v + (size_t)row * a.ldv;
    const int k0 = a.num_heads, v0 = a.num_heads + kv.kv_heads;  // the first key's and value's vector

    float x[AP_VECS<TYPE>][4], y[AP_VECS<TYPE>][4];
#pragma unroll
    for (int n = 0; n < AP_VECS<TYPE>; n++) {
        const int vec = first + n;
        const float *src = vec < k0 ? rq + vec * hd : vec < v0 ? rk + (vec - k0) * hd : rv + (vec - v0) * hd;
        if (live && vec < per_row) {
            load4(src + i0, a.vec, x[n]);
            load4(src + i1, a.vec, y[n]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) x[n][j] = y[n][j] = 0.f;
        }
    }
    int seq = 0, pos = -1;
    if (live) row_place(kv, b, row, seq, pos);
    bool ok = pos >= 0;
    float c[4], s[4];
    if (ok && rd > 0) {
        if (pos >= a.rope_rows) {
            paged_flag(kv, PAGED_BAD_POSITION);
            ok = false;
        } else if (turns) {
            const size_t at = (size_t)pos * (rd / 2) + 4 * l;
            load4(a.cos + at, a.vec, c);
            load4(a.sin + at, a.vec, s);
        }
    }
    // the row's slot in KV head 0, and its scale's place
    long long slot = -1, scale = -1;
    if (ok && first + AP_VECS<TYPE> > k0) {
        unsigned in_page;
        const int page = key_page(kv, b, seq, (unsigned)pos, in_page);
        if (page >= 0) {
            slot = row_offset(kv, page, 0, in_page);
            if constexpr (TYPE == KV_Q8) scale = scale_offset(kv, page, 0, in_page);
        } else if (page_index(kv, (unsigned)pos) < b.table_stride) {  // (a position past the table has its own flag)
            paged_flag(kv, PAGED_BAD_PAGE);
        }
    }
    if (a.q_norm || a.k_norm) {
#pragma unroll
        for (int n = 0; n < AP_VECS<TYPE>; n++) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) ss = __fmaf_rn(x[n][j], x[n][j], __fmaf_rn(y[n][j], y[n][j], ss));
#pragma unroll
            for (int o = LPV / 2; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
            const int vec = first + n;
            const float *w = vec < k0 ? a.q_norm : vec < v0 ? a.k_norm : nullptr;
            if (live && w) {
                const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)hd), a.eps)));
                float wx[4], wy[4];
                load4(w + i0, a.vec, wx);
                load4(w + i1, a.vec, wy);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[n][j] = __fmul_rn(__fmul_rn(x[n][j], r), wx[j]);
                    y[n][j] = __fmul_rn(__fmul_rn(y[n][j], r), wy[j]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < AP_VECS<TYPE>; n++) {
        const int vec = first + n;
        if (ok && turns && vec < v0) {
            if (split) {
#pragma unroll
                for (int j = 0; j < 4; j++) turn(x[n][j], y[n][j], c[j], s[j]);
            } else {
                turn(x[n][0], x[n][1], c[0], s[0]);
                turn(x[n][2], x[n][3], c[1], s[1]);
                turn(y[n][0], y[n][1], c[2], s[2]);
                turn(y[n][2], y[n][3], c[3], s[3]);
            }
        }
    }
    float top[AP_VECS<TYPE>];  // the vector's largest magnitude, NaN where it holds one
    if constexpr (TYPE == KV_Q8) {
#pragma unroll
        for (int n = 0; n < AP_VECS<TYPE>; n++) {
            top[n] = max3_abs(max3_abs(max3_abs(x[n][0], x[n][1], x[n][2]), x[n][3], y[n][0]),
                              max3_abs(y[n][1], y[n][2], y[n][3]), 0.f);
#pragma unroll
            for (int o = LPV / 2; o > 0; o >>= 1) top[n] = max3_abs(top[n], __shfl_xor_sync(0xffffffffu, top[n], o), 0.f);
        }
    }
    if (!live) return;
#pragma unroll
    for (int n = 0; n < AP_VECS<TYPE>; n++) {
        const int vec = first + n;
        if (vec >= per_row) break;
        if (vec < k0) {
            float *dst = a.q_out + (size_t)row * a.ldq_out + vec * hd;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[n][j] = ok ? x[n][j] : 0.f;
                y[n][j] = ok ? y[n][j] : 0.f;
            }
            if (a.vec) {
                *reinterpret_cast<float4 *>(dst + i0) = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
                *reinterpret_cast<float4 *>(dst + i1) = make_float4(y[n][0], y[n][1], y[n][2], y[n][3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) dst[i0 + j] = x[n][j], dst[i1 + j] = y[n][j];
            }
        } else if (slot >= 0) {
            const bool key = vec < v0;
            const long long above = (long long)(vec - (key ? k0 : v0)) * kv.page_size;  // rows of the heads before
            T *pool = reinterpret_cast<T *>(key ? kv.k : kv.v) + slot + above * hd;
            if constexpr (TYPE == KV_Q8) {
                const Q8Row r = q8_row(__float_as_uint(top[n]));
                const unsigned lo = q8_pack(x[n], r.up), hi = q8_pack(y[n], r.up);
                if (i1 == i0 + 4) {
                    *reinterpret_cast<uint2 *>(pool + i0) = make_uint2(lo, hi);
                } else {
                    *reinterpret_cast<unsigned *>(pool + i0) = lo;
                    *reinterpret_cast<unsigned *>(pool + i1) = hi;
                }
                if (l == 0)
                    *reinterpret_cast<float *>(reinterpret_cast<char *>(key ? kv.k : kv.v) + scale + above * 4) = r.scale;
            } else {
                KvElem<TYPE>::store4(pool + i0, x[n]);
                KvElem<TYPE>::store4(pool + i1, y[n]);
            }
        }
    }
}

template <int TYPE>
void append_typed(const KvView &kv, const BatchView &b, const AppendView &a, cudaStream_t s) {
    const uint64_t items = (uint64_t)b.num_rows * (unsigned)((a.num_heads + 2 * kv.kv_heads + AP_VECS<TYPE> - 1) / AP_VECS<TYPE>);
    auto go = [&](auto kernel, int lpv) {
        const uint64_t per = AP_THREADS / lpv;
        launch_kernel(kernel, dim3((unsigned)((items + per - 1) / per)), dim3(AP_THREADS), 0, s, TYPE == KV_Q8, kv, b, a);
    };
    if (kv.hd <= 32)
        go(paged_append_kernel<TYPE, 4>, 4);
    else if (kv.hd <= 64)
        go(paged_append_kernel<TYPE, 8>, 8);
    else
        go(paged_append_kernel<TYPE, 16>, 16);
}

// Rows of the cache as they were appended: a group of lanes (a power of two, 8
// elements each) takes the K and the V of one KV head of a row.  (8 x 4096 rows of 3
// heads of 64, 8-bit to f16, 38.5 MB: 15.2 us with the launch, 2.5 TB/s; two, three, four
// heads a group, for which the row's place is found once, 19.2, 17.4, 21.4.  What it
// waits for is a chain: the row's sequence, its page's id, the row.)
constexpr int RD_THREADS = 256;

template <int TYPE>
__device__ __forceinline__ void read8(const void *pool, long long at, long long scale, float (&x)[8]) {
    if constexpr (TYPE == KV_F32) {
        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(pool) + at);
        const float4 u = p[0], v = p[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else if constexpr (TYPE == KV_Q8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(reinterpret_cast<const char *>(pool) + at);
        const float f = scale_get(pool, scale);
        const unsigned w[2] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u};
#pragma unroll
        for (int j = 0; j < 8; j++)  // 2^23 + b + 128 is b + 128 under the exponent of 2^23
            x[j] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w[j >> 2], 0x4b000000u, 0x7440 | (j & 3))), 8388736.0f), f);
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(pool) + 2 * at);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float2 f;
            if constexpr (TYPE == KV_F16)
                f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
            else
                f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[j]));
            x[2 * j] = f.x, x[2 * j + 1] = f.y;
        }
    }
}
template <int OUT>
__device__ __forceinline__ void write8(void *out, size_t at, const float (&x)[8], bool vec) {
    using T = typename KvElem<OUT>::T;
    T *p = reinterpret_cast<T *>(out) + at;
    alignas(16) T y[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if constexpr (OUT == KV_F32)
            y[j] = x[j];
        else if constexpr (OUT == KV_F16)
            y[j] = __float2half_rn(x[j]);
        else
            y[j] = __float2bfloat16_rn(x[j]);
    }
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof y / 16; i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(y)[i];
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = y[j];
    }
}

template <int TYPE, int OUT>
__global__ void __launch_bounds__(RD_THREADS) paged_read_kernel(KvView kv, BatchView b, ReadView a, int lanes_log2) {
    pdl_wait();
    pdl_release();
    const unsigned item = (blockIdx.x * (unsigned)RD_THREADS + threadIdx.x) >> lanes_log2;  // below 2^32: the host's check
    const int l = threadIdx.x & ((1 << lanes_log2) - 1);
    const unsigned row = item / (unsigned)kv.kv_heads, head = item - row * (unsigned)kv.kv_heads;
    if (row >= (unsigned)b.num_rows || l * 8 >= kv.hd) return;
    int seq, pos;
    row_place(kv, b, (int)row, seq, pos);
    int page = -1;
    unsigned slot = 0;
    if (pos >= 0) page = key_page(kv, b, seq, (unsigned)pos, slot);
    const long long at = page < 0 ? 0 : row_offset(kv, page, (int)head, slot) + l * 8;
    const long long scale = page < 0 || TYPE != KV_Q8 ? 0 : scale_offset(kv, page, (int)head, slot);
    const size_t to = (size_t)head * kv.hd + l * 8;
    float k[8] = {}, v[8] = {};
    if (page >= 0 && a.k) read8<TYPE>(kv.k, at, scale, k);
    if (page >= 0 && a.v) read8<TYPE>(kv.v, at, scale, v);
    if (a.k) write8<OUT>(a.k, (size_t)row * a.ldk + to, k, a.vec);
    if (a.v) write8<OUT>(a.v, (size_t)row * a.ldv + to, v, a.vec);
}

template <int TYPE>
void read_typed(const KvView &kv, const BatchView &b, const ReadView &a, cudaStream_t s) {
    const int log2 = kv.hd <= 8 ? 0 : kv.hd <= 16 ? 1 : kv.hd <= 32 ? 2 : kv.hd <= 64 ? 3 : 4;
    const uint64_t threads = ((uint64_t)b.num_rows * kv.kv_heads) << log2;
    const unsigned grid = (unsigned)((threads + RD_THREADS - 1) / RD_THREADS);
    if (a.type == KV_F32)
        launch_kernel(paged_read_kernel<TYPE, KV_F32>, dim3(grid), dim3(RD_THREADS), 0, s, true, kv, b, a, log2);
    else if (a.type == KV_F16)
        launch_kernel(paged_read_kernel<TYPE, KV_F16>, dim3(grid), dim3(RD_THREADS), 0, s, true, kv, b, a, log2);
    else
        launch_kernel(paged_read_kernel<TYPE, KV_BF16>, dim3(grid), dim3(RD_THREADS), 0, s, true, kv, b, a, log2);
}

// Sequences that go on from others: CTA (i, y) makes sequence i's row of the
// table (y 0) and copies the used slots of its parent's last page, layers y *
// per_cta on, where i needs a page of its own.  A warp takes a (layer, K or V) at
// a time, its lanes 16-byte pieces of the used slots of all KV heads, four loads
// in flight: the pages lie scattered and hold 2 to 8 KB of a layer's keys.
constexpr int FK_THREADS = 128, FK_WARPS = FK_THREADS / 32, FK_PER = 2;

__global__ void __launch_bounds__(FK_THREADS) paged_fork_kernel(ForkPools pools, KvView kv, ForkView a, int layers, int per_cta,
                                                                int el) {
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int p = a.parent[i];
    if (p >= a.num_seqs) {
        if (tid == 0 && blockIdx.y == 0) paged_flag(kv, PAGED_BAD_ROWS);
        p = -1;
    }
    const bool table = blockIdx.y == 0 && a.table_out != nullptr;
    if (p < 0) {
        if (table) {
            for (int j = tid; j < a.stride; j += FK_THREADS) a.table_out[(size_t)i * a.stride + j] = -1;
            if (tid == 0) a.len_out[i] = 0;
            if (tid == 0 && a.taken) a.taken[i] = 0;
        }
        return;
    }
    // the first successor of a parent goes on in its pages
    int before = 0;
    for (int j = tid; j < i && !before; j += FK_THREADS) before = a.parent[j] == p;
    const int len = max(a.kv_len[p], 0);
    const unsigned tail = page_index(kv, (unsigned)len), used = (unsigned)len - tail * (unsigned)kv.page_size;
    const int32_t *old = a.table + (size_t)p * a.stride;
    const bool in_table = tail < (unsigned)a.stride;
    int source = in_table ? old[tail] : -1;
    int spare = a.spare ? a.spare[i] : -1;
    const bool first = !__syncthreads_or(before);
    if (tid == 0 && blockIdx.y == 0 && (tail > (unsigned)a.stride || (!in_table && used))) paged_flag(kv, PAGED_BAD_POSITION);
    const bool held = (unsigned)source < (unsigned)kv.num_pages;
    if (source >= 0 && !held && tid == 0 && blockIdx.y == 0) paged_flag(kv, PAGED_BAD_PAGE);
    // a page of its own: for the used slots that another goes on to fill, or for the next position
    const bool copies = !first && in_table && used && held;
    const bool wants = copies || (in_table && !used && (!first || source < 0));
    if (!wants) spare = -1;
    if ((unsigned)spare >= (unsigned)kv.num_pages) {
        if (tid == 0 && blockIdx.y == 0 && (spare >= 0 || copies)) paged_flag(kv, PAGED_BAD_PAGE);
        spare = -1;
    }
    if (table) {
        for (int j = tid; j < a.stride; j += FK_THREADS) {
            int id = first || (unsigned)j < tail ? old[j] : -1;
            if ((unsigned)j == tail && wants) id = spare;
            a.table_out[(size_t)i * a.stride + j] = id;
        }
        if (tid == 0) a.len_out[i] = len;
        if (tid == 0 && a.taken) a.taken[i] = wants && spare >= 0;
    }
    if (!copies || spare < 0) return;
    // pieces of 16 bytes, a slot's (a whole number) first: a page has fewer than 2^31, though 2^35 bytes
    const unsigned piece = (unsigned)(kv.hd * el) / 16u, chunks = used * piece;  // of a KV head's used slots
    const unsigned all = chunks * (unsigned)kv.kv_heads, gap = (unsigned)kv.page_size * piece - chunks;
    const uint64_t from = (uint64_t)source * kv.page_stride * el, to = (uint64_t)spare * kv.page_stride * el;
    const int end = min(layers, (int)(blockIdx.y + 1) * per_cta) * 2;
    for (int x = blockIdx.y * per_cta * 2 + warp; x < end; x += FK_WARPS) {
        char *pool = reinterpret_cast<char *>(x & 1 ? pools.v[x >> 1] : pools.k[x >> 1]);
        const uint4 *src = reinterpret_cast<const uint4 *>(pool + from);
        uint4 *dst = reinterpret_cast<uint4 *>(pool + to);
        for (unsigned e = lane; e < all; e += 128) {
            uint4 v[4];
            unsigned at[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const unsigned c = e + u * 32;
                at[u] = c + c / chunks * gap;
                if (c < all) v[u] = src[at[u]];
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (e + u * 32 < all) dst[at[u]] = v[u];
        }
        if (kv.type == KV_Q8)
            for (unsigned e = lane; e < used * (unsigned)kv.kv_heads; e += 32) {
                const unsigned h = e / used;
                const uint64_t at = kv.scale_at + ((uint64_t)h * (unsigned)kv.page_size + (e - h * used)) * 4u;
                *reinterpret_cast<float *>(pool + to + at) = *reinterpret_cast<const float *>(pool + from + at);
            }
    }
}

}  // namespace

void launch_paged_read(const KvView &kv, const BatchView &b, const ReadView &a, cudaStream_t s) {
    if (kv.type == KV_F32)
        read_typed<KV_F32>(kv, b, a, s);
    else if (kv.type == KV_F16)
        read_typed<KV_F16>(kv, b, a, s);
    else if (kv.type == KV_BF16)
        read_typed<KV_BF16>(kv, b, a, s);
    else
        read_typed<KV_Q8>(kv, b, a, s);
}

void launch_paged_fork(const ForkPools &pools, const KvView &kv, const ForkView &a, int layers, cudaStream_t s) {
    // two layers a CTA: a (layer, K or V) for each of its warps
    const int el = kv.type == KV_F32 ? 4 : kv.type == KV_Q8 ? 1 : 2, per_cta = FK_PER;
    launch_kernel(paged_fork_kernel, dim3((unsigned)a.num_new, (unsigned)((layers + per_cta - 1) / per_cta)), dim3(FK_THREADS), 0, s,
                  true, pools, kv, a, layers, per_cta, el);
}

void launch_paged_append(const KvView &kv, const BatchView &b, const AppendView &a, cudaStream_t s) {
    if (kv.type == KV_F32)
        append_typed<KV_F32>(kv, b, a, s);
    else if (kv.type == KV_F16)
        append_typed<KV_F16>(kv, b, a, s);
    else if (kv.type == KV_BF16)
        append_typed<KV_BF16>(kv, b, a, s);
    else
        append_typed<KV_Q8>(kv, b, a, s);
}

}  // namespace slm
