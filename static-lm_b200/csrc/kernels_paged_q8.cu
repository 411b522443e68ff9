// kernels_paged_q8.cu -- attention of several new rows per sequence (a prompt,
// or a chunk behind an earlier context) over 8-bit pages, on the tcgen05 tensor
// cores at f32 accuracy.
//
// A signed byte is exact in f16, so the copying warps turn bytes into f16 as they
// are and a row's scale is taken once: the key's by its column of scores, the
// value's by its column of weights.  q 2^e = q0 + q1 / 2^12 and the weights are
// two f16 parts each, 2 products for q.k and for w.v, as for f16 pages.  A value's
// scale enters the weights relative to a power of two at or above its tile's
// largest, which the f32 sums take back; a row whose sums come out far smaller (see
// Q8_RESULT_LEAST) is redone.  No chain of MMAs is longer than one
// key tile (the tensor core cuts each sum towards zero): every tile's w.v
// starts from zero and is added to the row's sums in registers.
//
// A CTA takes 256 rows of one (sequence, KV head), the query heads of the KV
// head side by side, as two streams of 128: warps 0-3 run the softmax of stream 0,
// a thread a row, warps 4-7 that of stream 1, warp 8 issues the MMAs of both,
// warps 9-11 bring keys and values.  The streams wait for nothing of each other,
// so one's arithmetic runs under the other's waits (w.v of its last tile and q.k
// of its next, 1000 of a tile's 3550 cycles at head_dim 64), and every key that is
// converted serves both.  8 x 4096 rows of 9 / 3 heads of 64: 530 us (292 TFLOP/s, two
// products for each; f16 pages 649); 16 chunks of up to 512 behind up to 8192, 32 / 8
// heads of 128: 742 us (345).  Neither issue (52 and 48 % of the cycles, about 14
// instructions a score and row) nor the tensor pipe (28 and 39 %) is full: a stream's
// warps wait for their own products, and the other stream's two warps an SM quarter
// cover a part of that; at head_dim 128 the copying warps are busy throughout, too.
#include "kernels.h"
#include "paged_tc.cuh"

namespace slm {

namespace {

constexpr unsigned PQ_TMEM_COLS = 512;

template <int HDP>
struct Q8Cfg {
    static constexpr int KT = 64;             // keys per tile: a thread holds a tile's scores in registers
    // Of which it works on 16 at a time, in a loop: code that is unrolled further leaves
    // the instruction cache.  (8 x 4096 rows of 9 / 3 heads of 64 and chunks of 32 / 8 of
    // 128, before q came by whole rows: 16 keys 541 and 765 us, 32 541 and 818, all 64 660
    // and 1073; now 530 and 742.)
    static constexpr int KC = 16;
    static constexpr bool Q_TMEM = HDP == 64;  // q's parts in TMEM (from shared memory an MMA of 64 columns takes 48 cycles, not 32)
    static constexpr int PRODUCERS = 96, THREADS = 384;
    static constexpr int R_LAUNCH = 168, R_SOFTMAX = HDP == 64 ? 208 : 200, R_OTHER = HDP == 64 ? 88 : 104;
    static_assert(256 * R_SOFTMAX + (THREADS - 256) * R_OTHER == THREADS * R_LAUNCH, "registers");
    static constexpr int QPART = 128 * HDP * 2;
    static constexpr int STREAM = 2 * QPART;  // q's parts, and after them the results, f32
    static constexpr int SLOT = KT * HDP * 2;  // k and v of even and of odd tiles, f16
    static constexpr int RAW = KT * HDP;       // the same as bytes
    static constexpr int A_KV = 2 * STREAM, A_RAW = A_KV + 4 * SLOT, BIG = A_RAW + 4 * RAW;
    // TMEM columns, of both streams: scores from 0 on, weights, q's parts, results
    static constexpr int T_W = 2 * KT, T_Q = 4 * KT, T_O = Q_TMEM ? T_Q + 128 : 256;
    static_assert(T_O + 2 * HDP <= (int)PQ_TMEM_COLS, "TMEM");
    // at least 120 KB: one CTA per SM, whose TMEM it takes whole
    static constexpr int SMALL = 3 * 1024, SMEM = (BIG > 120 * 1024 ? BIG : 120 * 1024) + SMALL;
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

// The small shared data, after the tiles.
struct Q8Shared {
    uint64_t full[4], empty[4], s_full[2], p_full[2], o_full[2], q_full[2], drain;
    long long off[64];        // byte offsets of the newest tile's keys
    alignas(16) float scale[4][2][64];  // of the keys and values of the newest 4 tiles
    unsigned valid[8][2];     // held keys of the newest 8 tiles
    float down[8];            // what their values' scales are relative to
    unsigned top[2];
    float most;               // the largest of all tiles' down
    unsigned taddr;
    int abort;
    // the CTA's work
    int seq, row0, rows, past, tile, found, bits;  // row0: first activation row of the sequence
};
static_assert(sizeof(Q8Shared) <= 3 * 1024 && offsetof(Q8Shared, scale) % 16 == 0 && offsetof(Q8Shared, off) % 8 == 0,
              "small shared data");

// A bounded wait; false once any wait of the CTA gave up.
__device__ __forceinline__ bool pq_wait(uint64_t *bar, unsigned parity, Q8Shared *sh, const KvView &kv) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_test(bar, parity)) {
        if (*(volatile int *)&sh->abort) return false;
        if (clock64() - t0 > WAIT_LIMIT) {
            *(volatile int *)&sh->abort = 1;
            paged_flag(kv, PAGED_WAIT_GAVE_UP);
            return false;
        }
    }
    return true;
}

// Bytes 0, 1 and 2, 3 of four signed ones as f16 pairs: 1024 + b + 128 is b + 128
// under an exponent byte of 0x64.
__device__ __forceinline__ uint2 bytes_f16(unsigned w) {
    const unsigned flipped = w ^ 0x80808080u;
    const unsigned lo = __byte_perm(flipped, 0x64646464u, 0x4140), hi = __byte_perm(flipped, 0x64646464u, 0x4342);
    uint2 r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(lo), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(hi), "r"(0x64806480u));
    return r;
}

template <int HDP>
__global__ void __launch_bounds__(Q8Cfg<HDP>::THREADS, 1) paged_rows_q8_kernel(KvView kv, BatchView b, PagedAttnView a, RowsPlan plan) {
    using Cfg = Q8Cfg<HDP>;
    using Range = WeightRange<KV_F16>;
    constexpr int KT = Cfg::KT, KC = Cfg::KC;
    extern __shared__ __align__(1024) unsigned char pq_smem[];
    Q8Shared *sh = reinterpret_cast<Q8Shared *>(pq_smem + Cfg::SMEM - Cfg::SMALL);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.num_heads / kv.kv_heads, hd = kv.hd;
    if (smem_addr(pq_smem) & 1023u) {  // the swizzled tiles need it
        if (tid == 0) paged_flag(kv, PAGED_WAIT_GAVE_UP);
        return;
    }
    pdl_release();
    zero_unowned_rows(kv, b, a, Cfg::THREADS);
    // this CTA's rows: blocks of 256 are counted from the last sequence's last
    // (the longest under the causal mask) to the first
    const int split = blockIdx.x % plan.splits;
    const int head = blockIdx.x / plan.splits % kv.kv_heads;
    const int index = blockIdx.x / plan.splits / kv.kv_heads;
    if (warp == 0) find_row_tile<8>(b, group, index, sh);
    __syncthreads();
    if (!sh->found) {
        if (tid == 0 && sh->bits) paged_flag(kv, sh->bits);
        return;
    }
    if (warp == 0) tc_alloc(&sh->taddr, PQ_TMEM_COLS);
    if (tid == 32) {
        for (int i = 0; i < 4; i++) {
            mbar_init(&sh->full[i], Cfg::PRODUCERS);
            mbar_init(&sh->empty[i], 1);
        }
        for (int x = 0; x < 2; x++) {
            mbar_init(&sh->s_full[x], 1);
            mbar_init(&sh->p_full[x], 4);
            mbar_init(&sh->o_full[x], 1);
            mbar_init(&sh->q_full[x], 4);
        }
        mbar_init(&sh->drain, 1);
        sh->abort = 0;
        sh->most = 0.f;
        mbar_fence_init();
    }
    const int seq = sh->seq, row0 = sh->row0, rows = sh->rows, tile = sh->tile;
    const int pos0 = b.kv_len[seq] - rows - sh->past;  // position of the sequence's first row
    // tokens of this block, and the list of keys any of them sees
    const unsigned flat0 = (unsigned)tile * 256u;
    const unsigned flat_end = (unsigned)rows * (unsigned)group;  // below 2^31: the host's check
    const int streams = flat_end - flat0 > 128u ? 2 : 1;
    const int tok0 = (int)(flat0 / (unsigned)group);
    int tok1 = (int)((flat0 + 255u) / (unsigned)group);
    tok1 = tok1 < rows ? tok1 : rows - 1;
    const SeenKeys keys = seen_keys(b, pos0 + tok0, pos0 + tok1, a.window, a.sinks);
    const int bits = sh->bits | (pos0 + tok1 >= b.cap ? PAGED_BAD_POSITION : 0);
    if (bits && tid == 0) paged_flag(kv, bits);
    const int all_tiles = (keys.n + KT - 1) / KT;
    const int per_split = (all_tiles + plan.splits - 1) / plan.splits;
    const int lo = split * per_split * KT;
    int hi = lo + per_split * KT;
    hi = hi < keys.n ? hi : keys.n;
    const int ntile = lo < hi ? (hi - lo + KT - 1) / KT : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (sh->taddr != 0) {  // never: all 512 columns start at column 0
        if (tid == 0) paged_flag(kv, PAGED_WAIT_GAVE_UP);
        __syncthreads();
        if (warp == 0) tc_dealloc(sh->taddr, PQ_TMEM_COLS);
        return;
    }

    // the softmax threads keep a tile's scores and the row's sums in registers:
    // they take some of the others'
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(Cfg::R_SOFTMAX));
        // ------------------------------------------------ q, softmax, output
        const int x = warp >> 2, r = tid & 127;  // stream, row of it
        if (x < streams) {
            const float sl2_all = __fmul_rn(a.scale, 1.44269504088896340736f);
            const unsigned flat = flat0 + (unsigned)(x * 128 + r);
            const int tok = (int)(flat / (unsigned)group), h = head * group + (int)(flat % (unsigned)group);
            const bool row_ok = tok < rows;
            const int row = row0 + (row_ok ? tok : 0);
            const int pos = row_ok ? pos0 + tok : -1;
            const unsigned t_lane = (unsigned)((warp & 3) * 32) << 16;
            const unsigned t_s = t_lane + (unsigned)(x * KT), t_w = t_lane + (unsigned)(Cfg::T_W + x * KT), t_o = t_lane + (unsigned)(Cfg::T_O + x * HDP);
            float sl2;
            {  // the row of q in two parts, scaled so that its largest element is near 2^15
                // It comes through the stream's shared memory, whole rows at a time, 16-byte chunk
                // c of row r at chunk c ^ (r & 7).  (Every thread its own row: 4400 to 9000
                // cycles of a CTA, since each load met 32 lines.)
                constexpr int LPR = HDP / 4, RPP = 32 / LPR;  // lanes a row, rows a pass
                unsigned char *const s_f = pq_smem + x * Cfg::STREAM + (warp & 3) * 32 * HDP * 4;
                const long long my_at = row_ok ? (long long)((size_t)row * a.ldq + (size_t)h * hd) : -1;
                if ((((uintptr_t)a.q | (a.ldq * 4)) & 15) == 0) {
#pragma unroll 4
                    for (int i = 0; i < 32; i += RPP) {
                        const int rr = i + lane / LPR, c = lane % LPR;
                        const long long at = __shfl_sync(0xffffffffu, my_at, rr);
                        const bool in = at >= 0 && c * 4 < hd;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(s_f + (rr * LPR + (c ^ (rr & 7))) * 16)),
                                     "l"(a.q + (in ? at + c * 4 : 0)), "r"(in ? 16u : 0u));
                    }
                } else {
#pragma unroll 4
                    for (int e = lane; e < 32 * HDP; e += 32) {
                        const int rr = e / HDP, d = e % HDP;
                        const long long at = __shfl_sync(0xffffffffu, my_at, rr);
                        const bool in = at >= 0 && d < hd;
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(
                                         smem_addr(s_f + (rr * LPR + ((d >> 2) ^ (rr & 7))) * 16 + (d & 3) * 4)),
                                     "l"(a.q + (in ? at + d : 0)), "r"(in ? 4u : 0u));
                    }
                }
                cp_async_commit();
                cp_async_wait<0>();
                __syncwarp();
                float f[HDP];  // (the row's sums are not yet in the registers)
#pragma unroll
                for (int c = 0; c < LPR; c++) {
                    const float4 t = *reinterpret_cast<const float4 *>(s_f + (lane * LPR + (c ^ (lane & 7))) * 16);
                    f[4 * c] = t.x, f[4 * c + 1] = t.y, f[4 * c + 2] = t.z, f[4 * c + 3] = t.w;
                }
                if constexpr (!Cfg::Q_TMEM) named_bar_sync(2 + x, 128);  // the parts go over other warps' rows
                unsigned top = 0;  // the bits of non-negative floats order as they do
#pragma unroll
                for (int d = 0; d < HDP; d++) top = max(top, __float_as_uint(fabsf(f[d])));
                int e = 141 - (int)(top >> 23);  // 2^14 <= top 2^e < 2^15
                e = top == 0 || top >= 0x7f800000u ? 0 : e > 120 ? 120 : e;
                const float up = __uint_as_float((unsigned)(127 + e) << 23);
                sl2 = __fmul_rn(sl2_all, __uint_as_float((unsigned)(127 - e) << 23));
#pragma unroll
                for (int d = 0; d < HDP; d += 32) {
                    unsigned part[2][16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        split2_f16(__fmul_rn(f[d + i], up), __fmul_rn(f[d + i + 1], up), part[0][i / 2], part[1][i / 2]);
                    }
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        if constexpr (Cfg::Q_TMEM) {
                            tmem_st16(t_lane + (unsigned)(Cfg::T_Q + x * 64 + n * 32 + d / 2), part[n]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<uint4 *>(pq_smem + x * Cfg::STREAM + n * Cfg::QPART + sw16_off(r, d / 8 + i, 128)) =
                                    make_uint4(part[n][4 * i], part[n][4 * i + 1], part[n][4 * i + 2], part[n][4 * i + 3]);
                        }
                    }
                }
                if constexpr (Cfg::Q_TMEM) {
                    tmem_wait_st();
                    tc_fence_before();
                } else {
                    fence_async_smem();
                }
                warp_arrive(&sh->q_full[x]);
            }
            // list positions this row sees: [0, sink_end) and [from, to)
            const int to = pos >= 0 ? pos - keys.low + keys.sinks + 1 : 0;
            const int sink_end = a.sinks < 0x7fffffffu ? (int)a.sinks : 0x7fffffff;
            int from = 0;
            if (a.window != 0 && pos >= 0 && (unsigned)pos >= a.window) from = pos - (int)a.window + 1 - keys.low + keys.sinks;
            float m = NO_MAX;
            uint64_t l2 = 0, acc[HDP / 2];  // pairs
#pragma unroll
            for (int i = 0; i < HDP / 2; i++) acc[i] = 0;
            bool ok = true;
            auto wait = [&](uint64_t *bar, int phase) {  // a warp goes on together: TMEM accesses are warp-wide
                ok = __all_sync(0xffffffffu, ok && pq_wait(bar, (unsigned)phase & 1u, sh, kv));
            };
            // adds tile j's w.v to the row's sums
            auto gather = [&](int j) {
                wait(&sh->o_full[x], j);
                if (!ok) return;
                tc_fence_after();
                const uint64_t down = pack2(sh->down[j & 7], sh->down[j & 7]);
#pragma unroll
                for (int c = 0; c < HDP; c += 32) {
                    float o[32];
                    tmem_ld32(t_o + c, o);
                    tmem_wait_ld();
                    pin32(o);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) acc[(c + i) / 2] = fma2(pack2(o[i], o[i + 1]), down, acc[(c + i) / 2]);
                }
            };
            const uint64_t sl2_2 = pack2(sl2, sl2);
            for (int j = 0; j < ntile; j++) {
                if (j > 0) gather(j - 1);  // which ends w.v of the weights whose place is taken next
                wait(&sh->s_full[x], j);
                if (!ok) break;
                tc_fence_after();
                const int i0 = lo + j * KT;
                const unsigned *valid = sh->valid[j & 7];
                const bool whole = i0 + KT <= to && i0 + KT <= hi && (i0 + KT <= sink_end || i0 >= from) &&
                                   (valid[0] & valid[1]) == 0xffffffffu;
                const bool masks = !__all_sync(0xffffffffu, whole);
                // The weights by the reference as it is, and the largest score under way:
                // where one has passed the reference by too much, all over again by a new
                // one.  (A pass for the maximum alone before each tile: 601 us, 8 x 4096 rows.)
                uint64_t l_before = l2;
                for (;;) {
                    const uint64_t minus_m = pack2(-m, -m);
                    float top = -INFINITY;
                    l2 = l_before;
#pragma unroll 1
                    for (int g = 0; g < KT / KC; g++) {
                        float v[KC];
                        tmem_ld16(t_s + g * KC, v);
                        const ulonglong2 *k_scales = reinterpret_cast<const ulonglong2 *>(sh->scale[j & 3][0] + g * KC);
                        const ulonglong2 *v_scales = reinterpret_cast<const ulonglong2 *>(sh->scale[j & 3][1] + g * KC);
                        uint64_t y[KC / 2];
#pragma unroll
                        for (int i = 0; i < KC / 2; i += 2) y[i] = k_scales[i / 2].x, y[i + 1] = k_scales[i / 2].y;
                        tmem_wait_ld();
                        pin16(v);
#pragma unroll
                        for (int i = 0; i < KC / 2; i++) y[i] = mul2(pack2(v[2 * i], v[2 * i + 1]), y[i]);
                        if (masks) {
                            // bit c: list position i0 + KC g + c is seen
                            auto below = [&](int end) -> unsigned {
                                const int n = end - (i0 + g * KC);
                                return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
                            };
                            const unsigned seen = below(to) & (below(sink_end) | ~below(from)) & (valid[g * KC / 32] >> (g * KC % 32));
#pragma unroll
                            for (int i = 0; i < KC / 2; i++) {
                                float s0, s1;
                                unpack2(y[i], s0, s1);
                                y[i] = pack2(seen & (1u << (2 * i)) ? s0 : -INFINITY, seen & (1u << (2 * i + 1)) ? s1 : -INFINITY);
                            }
                        }
                        unsigned w[2][KC / 2];
#pragma unroll
                        for (int i = 0; i < KC / 2; i += 2) {
                            const ulonglong2 vs = v_scales[i / 2];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                float e0, e1;
                                unpack2(y[i + u], e0, e1);
                                top = fmaxf(top, fmaxf(e0, e1));
                                unpack2(fma2(y[i + u], sl2_2, minus_m), e0, e1);
                                const uint64_t e = pack2(exp2_approx(e0), exp2_approx(e1));
                                l2 = add2(l2, e);
                                unpack2(mul2(e, u ? vs.y : vs.x), e0, e1);
                                split2_f16(e0, e1, w[0][i + u], w[1][i + u]);
                            }
                        }
                        // part n of KC keys at column n KC / 2
                        tmem_st8(t_w + g * KC, w[0]);
                        tmem_st8(t_w + g * KC + KC / 2, w[1]);
                    }
                    top = __fmul_rn(top, sl2);
                    const bool move = top > m + Range::rescale;
                    if (!__any_sync(0xffffffffu, move)) break;
                    if (move) {
                        const float to_m = __fsub_rn(top, Range::margin);
                        const float f = exp2_approx(__fsub_rn(m, to_m));
                        m = to_m;
                        const uint64_t f2 = pack2(f, f);
                        l_before = mul2(l_before, f2);
#pragma unroll
                        for (int i = 0; i < HDP / 2; i++) acc[i] = mul2(acc[i], f2);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(&sh->p_full[x]);
            }
            if (ok && ntile > 0) gather(ntile - 1);
            // (a warp that broke off leaves the others' waits to give up: all meet here)
            if (!named_bar_or(2 + x, 128, !ok)) {
                float l, l_odd;
                unpack2(l2, l, l_odd);
                l = __fadd_rn(l, l_odd);
                const bool split_up = plan.splits > 1;
                const float inv = split_up ? 1.0f : l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
                // Once a reference was set, l is 2^margin or more, but for scores past
                // 2^24, of which x - m keeps the bits that m, rounded, has lost.
                bool finite = fabsf(l) < INFINITY && (m == NO_MAX || l >= Range::least);
                // every product of the stream is complete: the results go through its
                // shared memory, 16-byte chunk c of row r at chunk c ^ (r & 7), to whole rows
                float4 *s_o = reinterpret_cast<float4 *>(pq_smem + x * Cfg::STREAM + (warp & 3) * 32 * HDP * 4);
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < HDP; i += 4) {
                    float y[4];
                    unpack2(acc[i / 2], y[0], y[1]);
                    unpack2(acc[i / 2 + 1], y[2], y[3]);
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        y[u] = __fmul_rn(y[u], inv);
                        if (i < hd) finite = finite && fabsf(y[u]) < INFINITY, largest = fmaxf(largest, fabsf(y[u]));
                    }
                    s_o[lane * (HDP / 4) + ((i / 4) ^ (lane & 7))] = make_float4(y[0], y[1], y[2], y[3]);
                }
                finite = finite && largest >= __fmul_rn(__fmul_rn(sh->most, Q8_RESULT_LEAST), l == 0.f ? 0.f : inv);
                if (split_up && row_ok)
                    plan.part_ml[((size_t)row * a.num_heads + h) * plan.splits + split] = make_float2(m, l);
                __syncwarp();
                const bool vec = split_up || (((uintptr_t)a.out | (a.ldo * 4)) & 15) == 0;
                constexpr int LPR = HDP / 4, RPP = 32 / LPR;  // lanes a row, rows a pass
                const int c = lane % LPR;
                const long long my_at = !row_ok ? -1
                                        : split_up ? (long long)((((size_t)row * a.num_heads + h) * plan.splits + split) * hd)
                                                   : (long long)((size_t)row * a.ldo + (size_t)h * hd);
                float *const to_base = (split_up ? plan.part_o : a.out) + c * 4;
#pragma unroll 2
                for (int i = 0; i < 32; i += RPP) {
                    const int rr = i + lane / LPR;
                    const long long at = __shfl_sync(0xffffffffu, my_at, rr);
                    if (at < 0 || c * 4 >= hd) continue;
                    float *dst = to_base + at;
                    const float4 y = s_o[rr * LPR + (c ^ (rr & 7))];
                    if (vec)
                        *reinterpret_cast<float4 *>(dst) = y;
                    else
                        dst[0] = y.x, dst[1] = y.y, dst[2] = y.z, dst[3] = y.w;
                }
                // rows that met a scale that is not finite or a large key's, scores so large, or
                // values beside which their own do not show, once the warp's first results are written
                __syncwarp();
                unsigned redo = __ballot_sync(0xffffffffu, row_ok && !finite);
                while (redo) {
                    const int who = __ffs(redo) - 1;
                    redo &= redo - 1;
                    const int rrow = __shfl_sync(0xffffffffu, row, who), rh = __shfl_sync(0xffffffffu, h, who);
                    const int rfrom = __shfl_sync(0xffffffffu, from, who), rto = __shfl_sync(0xffffffffu, to, who);
                    const RowState st = attend_row<KV_Q8>(kv, b, seq, head, a.q + (size_t)rrow * a.ldq + (size_t)rh * hd, sl2_all,
                                                          keys, lo, hi, rfrom, sink_end, rto);
                    const size_t at = ((size_t)rrow * a.num_heads + rh) * plan.splits + split;
                    float *d = split_up ? plan.part_o + at * hd : a.out + (size_t)rrow * a.ldo + (size_t)rh * hd;
                    const float div = split_up ? 1.0f : st.l;
#pragma unroll
                    for (int c4 = 0; c4 < 4; c4++)
                        if (lane + 32 * c4 < hd) d[lane + 32 * c4] = div == 0.f ? 0.f : __fdiv_rn(st.acc[c4], div);
                    if (split_up && lane == 0) plan.part_ml[at] = make_float2(st.m, st.l);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Cfg::R_OTHER));
    }
    if (warp < 8) {
    } else if (warp == 8) {
        // --------------------------------------------------------- the MMAs
        if (ntile > 0) {
            constexpr unsigned idesc_s = umma_idesc_f16(false, 128, KT, false);
            const unsigned idesc_o = umma_idesc_f16(false, 128, hd, true);
            const unsigned a_q = smem_addr(pq_smem), a_kv = a_q + Cfg::A_KV;
            bool ok = true;
            auto wait = [&](uint64_t *bar, int phase) {  // the warp goes on together
                ok = __all_sync(0xffffffffu, ok && pq_wait(bar, (unsigned)phase & 1u, sh, kv));
                tc_fence_after();
            };
            // A descriptor is a base's low word plus a constant (in 16 bytes; no carry: the
            // address has 14 bits there).  The base is made anew for every tile, else
            // all the descriptors are kept, more than the registers hold.
            auto plus = [](unsigned base, unsigned bytes, uint64_t of) -> uint64_t {
                return (of & 0xffffffff00000000ull) | (base + (bytes >> 4));
            };
            auto base_of = [](uint64_t desc) -> unsigned {
                unsigned lo = (unsigned)desc;
                asm volatile("" : "+r"(lo));
                return lo;
            };
            // k of slot parity P, stream X; the second parts' products first
            auto scores = [&](auto parity, auto stream) {
                constexpr int P = decltype(parity)::value, X = decltype(stream)::value;
                const uint64_t k_desc = umma_desc_sw128(a_kv + 2 * P * Cfg::SLOT), q_desc = umma_desc_sw128(a_q + X * Cfg::STREAM);
                const unsigned k_base = base_of(k_desc), q_base = base_of(q_desc);
#pragma unroll
                for (int i = 1; i >= 0; i--)
#pragma unroll
                    for (int ks = 0; ks < HDP / 16; ks++) {
                        const uint64_t bd = plus(k_base, (ks >> 2) * KT * 128 + (ks & 3) * 32, k_desc);
                        if constexpr (Cfg::Q_TMEM) {
                            const unsigned at = Cfg::T_Q + X * 64 + i * 32 + ks * 8;
                            if (i == 0 && ks == 0)
                                tc_mma_f16_ta_onto_part2(X * KT, at, bd, idesc_s);
                            else
                                tc_mma_f16_ta(X * KT, at, bd, idesc_s, i == 0 || ks > 0);
                        } else {
                            const uint64_t ad = plus(q_base, i * Cfg::QPART + (ks >> 2) * 128 * 128 + (ks & 3) * 32, q_desc);
                            if (i == 0 && ks == 0)
                                tc_mma_f16_onto_part2(X * KT, ad, bd, idesc_s);
                            else
                                tc_mma_f16(X * KT, ad, bd, idesc_s, i == 0 || ks > 0);
                        }
                    }
                tc_commit_elected(&sh->s_full[X]);
            };
            auto values = [&](auto parity, auto stream) {
                constexpr int P = decltype(parity)::value, X = decltype(stream)::value;
                constexpr unsigned d = Cfg::T_O + X * HDP;
                const uint64_t v_desc = umma_desc_sw128_mn(a_kv + (2 * P + 1) * Cfg::SLOT, KT * 128);
                const unsigned v_base = base_of(v_desc);
#pragma unroll
                for (int i = 1; i >= 0; i--)
#pragma unroll
                    for (int ks = 0; ks < KT / 16; ks++) {
                        const unsigned at = Cfg::T_W + X * KT + ks * KC + i * (KC / 2);
                        const uint64_t bd = plus(v_base, ks * 2048, v_desc);
                        if (i == 0 && ks == 0)
                            tc_mma_f16_ta_onto_part2(d, at, bd, idesc_o);
                        else
                            tc_mma_f16_ta(d, at, bd, idesc_o, i == 0 || ks > 0);
                    }
                tc_commit_elected(&sh->o_full[X]);
            };
            const std::integral_constant<int, 0> zero{};
            const std::integral_constant<int, 1> one{};
            // w.v of tile j, then q.k of tile j + 1 in the place of the scores that the
            // weights were made of, stream by stream
            auto step = [&](auto parity, int j) {
                constexpr int P = decltype(parity)::value;
                const std::integral_constant<int, 1 - P> other{};
                const bool more = j + 1 < ntile;
                wait(&sh->full[2 * P + 1], j >> 1);
                wait(&sh->p_full[0], j);
                fence_async_elected();
                if (!ok) return;
                values(parity, zero);
                if (more) {
                    wait(&sh->full[2 * (1 - P)], (j + 1) >> 1);
                    fence_async_elected();
                    if (!ok) return;
                    scores(other, zero);
                }
                if (streams == 2) {
                    wait(&sh->p_full[1], j);
                    if (!ok) return;
                    values(parity, one);
                }
                tc_commit_elected(&sh->empty[2 * P + 1]);
                if (more) {
                    if (streams == 2) scores(other, one);
                    tc_commit_elected(&sh->empty[2 * (1 - P)]);
                }
            };
            wait(&sh->q_full[0], 0);
            wait(&sh->full[0], 0);
            fence_async_elected();
            if (ok) scores(zero, zero);
            if (streams == 2) {
                wait(&sh->q_full[1], 0);
                if (ok) scores(zero, one);
            }
            if (ok) tc_commit_elected(&sh->empty[0]);
            for (int j = 0; j < ntile && ok; j += 2) {
                step(zero, j);
                if (j + 1 < ntile && ok) step(one, j + 1);
            }
            // what was issued has to end before the TMEM is freed
            tc_commit_elected(&sh->drain);
            const long long t0 = clock64();
            while (!mbar_test(&sh->drain, 0) && clock64() - t0 < WAIT_LIMIT) {
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------- keys and values to slots
        const int p = tid - 9 * 32;
        constexpr int CH = HDP / 16;                // 16-byte chunks of a row
        constexpr int RSTEP = Cfg::PRODUCERS / CH;  // rows a pass: 24 or 12
        constexpr int PASSES = (KT + RSTEP - 1) / RSTEP;
        static_assert(KC == 16, "an MMA's keys");
        static_assert(Cfg::PRODUCERS % CH == 0 && RSTEP % 4 == 0, "a thread keeps its chunk");
        const int c = p % CH, r_first = p / CH;
        const bool in_row = c * 16 < hd;
        bool ok = true;
        // Key p of a tile: its page id is on its way for a tile while that of the
        // tile before is made offsets, whose scales are on theirs.
        struct Id {
            int page;
            unsigned slot;
        };
        struct At {
            long long row;  // byte offset in the pools, -1 for none
            float k_scale, v_scale;
        };
        auto look = [&](int j) -> Id {
            const int at = lo + j * KT + p;
            if (p >= KT || at >= hi) return Id{-1, 0};  // (every list position is below the table's end)
            const unsigned key = (unsigned)keys.key(at), pi = page_index(kv, key);
            return Id{(int)ldg_now(b.table + (size_t)seq * b.table_stride + pi), key - pi * (unsigned)kv.page_size};
        };
        auto find = [&](Id id) -> At {
            if ((unsigned)id.page >= (unsigned)kv.num_pages) {
                if (id.page >= 0) paged_flag(kv, PAGED_BAD_PAGE);
                return At{-1, 0.f, 0.f};
            }
            const long long s = scale_offset(kv, id.page, head, id.slot);
            return At{row_offset(kv, id.page, head, id.slot), __uint_as_float(ldg_now(reinterpret_cast<const char *>(kv.k) + s)),
                      __uint_as_float(ldg_now(reinterpret_cast<const char *>(kv.v) + s))};
        };
        // tile j's bytes, by the thread that will turn them into f16
        auto copy = [&](int j) {
            const unsigned raw = smem_addr(pq_smem) + Cfg::A_RAW + (j & 1) * 2 * Cfg::RAW + p * 16;
#pragma unroll
            for (int n = 0; n < PASSES; n++) {
                const int row = r_first + n * RSTEP;
                if (row >= KT) break;
                const long long o = sh->off[row];
                const bool in = o >= 0 && in_row;
                const long long at = in ? o + c * 16 : 0;
#pragma unroll
                for (int i = 0; i < 2; i++)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(raw + i * Cfg::RAW + n * Cfg::PRODUCERS * 16),
                                 "l"(reinterpret_cast<const char *>(i ? kv.v : kv.k) + at), "r"(in ? 16u : 0u));
            }
            cp_async_commit();
        };
        auto convert = [&](int j, int i) {  // k (0) or v (1) of tile j
            const int s = 2 * (j & 1) + i;
            if (j >= 2) ok = pq_wait(&sh->empty[s], (unsigned)((j >> 1) - 1) & 1u, sh, kv);
            if (!ok) return;
            const unsigned char *raw = pq_smem + Cfg::A_RAW + ((j & 1) * 2 + i) * Cfg::RAW + p * 16;
            unsigned char *dst = pq_smem + Cfg::A_KV + s * Cfg::SLOT;
            uint4 w[PASSES];
#pragma unroll
            for (int n = 0; n < PASSES; n++)
                if (r_first + n * RSTEP < KT) w[n] = *reinterpret_cast<const uint4 *>(raw + n * Cfg::PRODUCERS * 16);
#pragma unroll
            for (int n = 0; n < PASSES; n++) {
                const int row = r_first + n * RSTEP;
                if (row >= KT) break;
                const uint2 b0 = bytes_f16(w[n].x), b1 = bytes_f16(w[n].y), b2 = bytes_f16(w[n].z), b3 = bytes_f16(w[n].w);
                *reinterpret_cast<uint4 *>(dst + sw16_off(row, 2 * c, KT)) = make_uint4(b0.x, b0.y, b1.x, b1.y);
                *reinterpret_cast<uint4 *>(dst + sw16_off(row, 2 * c + 1, KT)) = make_uint4(b2.x, b2.y, b3.x, b3.y);
            }
            fence_async_smem();
            mbar_arrive(&sh->full[s]);
        };
        At next = find(look(0));
        Id ahead = look(1);
        for (int j = 0; j < ntile && ok; j++) {
            // tile j's offsets and scales for all, its copies on their way, then the next tile's look-ups
            if (warp < 11) {
                const int w = warp - 9;
                sh->off[p] = next.row;
                const unsigned held = __ballot_sync(0xffffffffu, next.row >= 0);
                const unsigned bits_v = __float_as_uint(fabsf(next.v_scale));
                const unsigned top = __reduce_max_sync(0xffffffffu, bits_v < 0x7f800000u ? bits_v : 0u);
                if (lane == 0) sh->valid[j & 7][w] = held, sh->top[w] = top;
            }
            named_bar_sync(1, Cfg::PRODUCERS);
            copy(j);
            if (warp < 11) {
                // 2^e above the tile's largest scale of a value that is finite
                const unsigned top = max(sh->top[0], sh->top[1]);
                const int e = min(max((int)(top >> 23) - 126, -125), 126);
                // (NaN: the rows that see the key are redone)
                sh->scale[j & 3][0][p] = q8_large_key(q8_above_limit(next.k_scale)) ? __uint_as_float(0x7fc00000u) : next.k_scale;
                sh->scale[j & 3][1][p] = __fmul_rn(next.v_scale, __uint_as_float((unsigned)(127 - e) << 23));
                if (p == 0) {
                    const float down = top != 0 ? __uint_as_float((unsigned)(127 + e) << 23) : 0.f;
                    sh->down[j & 7] = down;
                    sh->most = fmaxf(sh->most, down);
                }
            }
            next = find(ahead);
            ahead = look(j + 2);
            if (j > 0) {
                cp_async_wait<1>();
                convert(j - 1, 0);
                if (ok) convert(j - 1, 1);
            }
            ok = !named_bar_or(1, Cfg::PRODUCERS, !ok);
        }
        cp_async_wait<0>();
        if (ok && ntile > 0) {
            convert(ntile - 1, 0);
            if (ok) convert(ntile - 1, 1);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tc_dealloc(0, PQ_TMEM_COLS);
}

template <int HDP>
void go(const KvView &kv, const BatchView &b, const PagedAttnView &a, const RowsPlan &plan, cudaStream_t s) {
    static SmemOptIn opt;
    opt(paged_rows_q8_kernel<HDP>, Q8Cfg<HDP>::SMEM);
    const unsigned grid = (unsigned)(plan.tiles * kv.kv_heads * plan.splits);
    launch_kernel(paged_rows_q8_kernel<HDP>, dim3(grid), dim3(Q8Cfg<HDP>::THREADS), Q8Cfg<HDP>::SMEM, s, false, kv, b, a, plan);
}

}  // namespace

void launch_paged_rows_q8(const KvView &kv, const BatchView &b, const PagedAttnView &a, const RowsPlan &plan, cudaStream_t s) {
    kv.hd <= 64 ? go<64>(kv, b, a, plan, s) : go<128>(kv, b, a, plan, s);
}

}  // namespace slm
