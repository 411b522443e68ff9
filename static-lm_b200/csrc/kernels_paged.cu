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

// LPV lanes (a power of two, 8 elements each) per head vector; the vectors of
// a row are its query heads, its key heads, then its value heads.
//   norm:  y = x * (1 / sqrt(sum(x^2) / head_dim + eps)) * w      (q and k)
//   turn:  (a, b) -> (a cos - b sin, a sin + b cos)                (q and k)
// with (a, b) neighbours, or the two halves of the first rotary_dim elements.
// Every product and sum is rounded on its own, so that the rotation gives the
// bits of slm_apply_rope_cached.
//
// Bound by memory: 8 bytes in and out per query element, 4 + the page's type
// per key and value element.  A thread's loads, its row's place (a search in
// row_start, the length, the page id) and the two table rows are a chain of
// latencies, so the registers are held to 32 for 64 warps an SM (40 registers:
// 53.3 us, 32: 51.2 us for 8 x 4096 rows of 9 + 3 + 3 heads of 64, f16 pages,
// cold: 4.6 TB/s of the 6.5 a copy reaches; single rows are a launch, 7 us
// with the call).
template <int TYPE, int LPV>
__global__ void __launch_bounds__(AP_THREADS, 8) paged_append_kernel(KvView kv, BatchView b, AppendView a) {
    using T = typename KvElem<TYPE>::T;
    const int l = threadIdx.x % LPV, hd = kv.hd;
    const int per_row = a.num_heads + 2 * kv.kv_heads;
    const unsigned item = blockIdx.x * (AP_THREADS / LPV) + threadIdx.x / LPV;  // below 2^32: the host's check
    const unsigned its_row = item / (unsigned)per_row;
    const bool live = its_row < (unsigned)b.num_rows && l * 8 < hd;
    const int row = live ? (int)its_row : 0;
    const int vec = live ? (int)(item - its_row * (unsigned)per_row) : 0;
    // kind 0 = query head, 1 = key head, 2 = value head
    const int kind = vec < a.num_heads ? 0 : vec < a.num_heads + kv.kv_heads ? 1 : 2;
    const int head = kind == 0 ? vec : kind == 1 ? vec - a.num_heads : vec - a.num_heads - kv.kv_heads;
    const float *src = kind == 0   ? a.q + (size_t)row * a.ldq
                       : kind == 1 ? a.k + (size_t)row * a.ldk
                                   : a.v + (size_t)row * a.ldv;
    const int rd = a.rotary_dim;
    const bool turned = kind != 2 && 8 * l < rd;
    const bool split = turned && a.halves;
    const int i0 = split ? 4 * l : 8 * l, i1 = split ? rd / 2 + 4 * l : 8 * l + 4;

    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        load4(src + (size_t)head * hd + i0, a.vec, x);
        load4(src + (size_t)head * hd + i1, a.vec, y);
    }
    int seq = 0, pos = -1;
    if (live) row_place(b, row, seq, pos);

    const float *w = kind == 0 ? a.q_norm : a.k_norm;
    if (kind == 2) w = nullptr;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) ss = __fmaf_rn(x[j], x[j], __fmaf_rn(y[j], y[j], ss));
#pragma unroll
    for (int o = LPV / 2; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
    if (!live) return;
    if (w) {
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)hd), a.eps)));
        float wx[4], wy[4];
        load4(w + i0, a.vec, wx);
        load4(w + i1, a.vec, wy);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = __fmul_rn(__fmul_rn(x[j], r), wx[j]);
            y[j] = __fmul_rn(__fmul_rn(y[j], r), wy[j]);
        }
    }
    bool ok = pos >= 0;
    if (ok && turned && pos >= a.rope_rows) {
        paged_flag(kv, PAGED_BAD_POSITION);
        ok = false;
    }
    if (ok && turned) {
        float c[4], s[4];
        const size_t at = (size_t)pos * (rd / 2) + 4 * l;
        load4(a.cos + at, a.vec, c);
        load4(a.sin + at, a.vec, s);
        if (split) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = x[j], q = y[j];
                x[j] = __fsub_rn(__fmul_rn(p, c[j]), __fmul_rn(q, s[j]));
                y[j] = __fadd_rn(__fmul_rn(p, s[j]), __fmul_rn(q, c[j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float p = x[2 * j], q = x[2 * j + 1];
                x[2 * j] = __fsub_rn(__fmul_rn(p, c[j]), __fmul_rn(q, s[j]));
                x[2 * j + 1] = __fadd_rn(__fmul_rn(p, s[j]), __fmul_rn(q, c[j]));
                p = y[2 * j], q = y[2 * j + 1];
                y[2 * j] = __fsub_rn(__fmul_rn(p, c[j + 2]), __fmul_rn(q, s[j + 2]));
                y[2 * j + 1] = __fadd_rn(__fmul_rn(p, s[j + 2]), __fmul_rn(q, c[j + 2]));
            }
        }
    }
    if (kind == 0) {
        float *dst = a.q_out + (size_t)row * a.ldq_out + (size_t)head * hd;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = ok ? x[j] : 0.f;
            y[j] = ok ? y[j] : 0.f;
        }
        if (a.vec) {
            *reinterpret_cast<float4 *>(dst + i0) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(dst + i1) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) dst[i0 + j] = x[j], dst[i1 + j] = y[j];
        }
        return;
    }
    if (!ok) return;
    const long long off = key_offset(kv, b, seq, (unsigned)pos, head);
    if (off < 0) {
        paged_flag(kv, PAGED_BAD_PAGE);
        return;
    }
    T *pool = reinterpret_cast<T *>(kind == 1 ? kv.k : kv.v) + off;
    KvElem<TYPE>::store4(pool + i0, x);
    KvElem<TYPE>::store4(pool + i1, y);
}

template <int TYPE>
void append_typed(const KvView &kv, const BatchView &b, const AppendView &a, cudaStream_t s) {
    const uint64_t items = (uint64_t)b.num_rows * (unsigned)(a.num_heads + 2 * kv.kv_heads);
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
