// kernels_paged.cu -- the paged key/value cache: new keys and values into
// their pages with the per-head RMSNorm and the position rotation applied on
// the way.
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
// launch's time.
constexpr int AP_VECS = 3;

template <int TYPE, int LPV>
__global__ void __launch_bounds__(AP_THREADS, 4) paged_append_kernel(KvView kv, BatchView b, AppendView a) {
    using T = typename KvElem<TYPE>::T;
    const int l = threadIdx.x % LPV, hd = kv.hd;
    const int per_row = a.num_heads + 2 * kv.kv_heads, parts = (per_row + AP_VECS - 1) / AP_VECS;
    const unsigned item = blockIdx.x * (AP_THREADS / LPV) + threadIdx.x / LPV;  // below 2^32: the host's check
    const unsigned its_row = item / (unsigned)parts;
    const bool live = its_row < (unsigned)b.num_rows && l * 8 < hd;
    const int row = live ? (int)its_row : 0;
    const int first = live ? (int)(item - its_row * (unsigned)parts) * AP_VECS : 0;
    const int rd = a.rotary_dim;
    const bool turns = 8 * l < rd;          // this lane's elements of q and k are rotated,
    const bool split = turns && a.halves;   // as pairs half of rotary_dim apart
    const int i0 = split ? 4 * l : 8 * l, i1 = split ? rd / 2 + 4 * l : 8 * l + 4;
    const float *const rq = a.q + (size_t)row * a.ldq, *const rk = a.k + (size_t)row * a.ldk,
                *const rv = a.v + (size_t)row * a.ldv;
    const int k0 = a.num_heads, v0 = a.num_heads + kv.kv_heads;  // the first key's and value's vector

    float x[AP_VECS][4], y[AP_VECS][4];
#pragma unroll
    for (int n = 0; n < AP_VECS; n++) {
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
    // the row's slot in KV head 0
    long long slot = -1;
    if (ok && first + AP_VECS > k0) {
        slot = key_offset(kv, b, seq, (unsigned)pos, 0);
        // (a position past the table has its own flag)
        if (slot < 0 && page_index(kv, (unsigned)pos) < b.table_stride) paged_flag(kv, PAGED_BAD_PAGE);
    }
    if (a.q_norm || a.k_norm) {
#pragma unroll
        for (int n = 0; n < AP_VECS; n++) {
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
    if (!live) return;
#pragma unroll
    for (int n = 0; n < AP_VECS; n++) {
        const int vec = first + n;
        if (vec >= per_row) break;
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
            T *pool = reinterpret_cast<T *>(key ? kv.k : kv.v) + slot + (long long)(vec - (key ? k0 : v0)) * kv.page_size * hd;
            KvElem<TYPE>::store4(pool + i0, x[n]);
            KvElem<TYPE>::store4(pool + i1, y[n]);
        }
    }
}

template <int TYPE>
void append_typed(const KvView &kv, const BatchView &b, const AppendView &a, cudaStream_t s) {
    const uint64_t items = (uint64_t)b.num_rows * (unsigned)((a.num_heads + 2 * kv.kv_heads + AP_VECS - 1) / AP_VECS);
    auto go = [&](auto kernel, int lpv) {
        const uint64_t per = AP_THREADS / lpv;
        kernel<<<(unsigned)((items + per - 1) / per), AP_THREADS, 0, s>>>(kv, b, a);
    };
    if (kv.hd <= 32)
        go(paged_append_kernel<TYPE, 4>, 4);
    else if (kv.hd <= 64)
        go(paged_append_kernel<TYPE, 8>, 8);
    else
        go(paged_append_kernel<TYPE, 16>, 16);
}

}  // namespace

void launch_paged_append(const KvView &kv, const BatchView &b, const AppendView &a, cudaStream_t s) {
    if (kv.type == KV_F32)
        append_typed<KV_F32>(kv, b, a, s);
    else if (kv.type == KV_F16)
        append_typed<KV_F16>(kv, b, a, s);
    else
        append_typed<KV_BF16>(kv, b, a, s);
}

}  // namespace slm
