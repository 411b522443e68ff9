// kernels_paged_decode.cu -- attention of one new row per sequence over the
// paged cache: the length split over CTAs, a warp's online softmax over its
// own keys, the partial results joined by a second small launch.
//
// With x_j = scale log2(e) q.k_j and any reference m,
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),
// so each warp keeps (m, l, o) over the keys it has read, and two such
// triples join as m = max, l = sum of l_i 2^(m_i - m), o alike.
#include "async.cuh"
#include "kernels.h"

namespace slm {

namespace {

constexpr int PD_WARPS = 4;
constexpr int PD_THREADS = PD_WARPS * 32;
constexpr int PD_STAGES = 2;  // 64 KB a CTA: three CTAs an SM (three stages and two CTAs: 8 % slower)
constexpr int PD_PASSES = 8;               // 512-byte passes per K (or V) tile
constexpr int PD_TILE = PD_PASSES * 512;   // bytes of a warp's K (or V) tile

// CTAs of g query heads that an SM holds: by shared memory, and by registers.
__host__ __device__ constexpr int ctas_per_sm(int g) { return g <= 4 ? 3 : 2; }

__device__ __forceinline__ void cp_async16_zfill(unsigned dst, const void *src, unsigned bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}

// The 16 bytes of one lane as f32 pairs.
__device__ __forceinline__ void load_chunk(unsigned a, uint64_t (&x)[2]) {
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(x[0]), "=l"(x[1]) : "r"(a));
}

// What the two kernels share of a CTA's work: keys [lo, hi) of the list that
// the row of sequence `seq` sees, KV head `head`, ng query heads from h0 on.
struct DecodeWork {
    int split, seq, head, h0, ng, lo, hi;
    SeenKeys keys;
};
__device__ __forceinline__ bool decode_work(const KvView &kv, const BatchView &b, const PagedAttnView &a,
                                            const DecodePlan &plan, DecodeWork &w) {
    w.split = blockIdx.x % plan.splits;
    int unit = blockIdx.x / plan.splits;
    const int hg = unit % plan.head_groups;
    unit /= plan.head_groups;
    w.head = unit % kv.kv_heads, w.seq = unit / kv.kv_heads;
    const int group = a.num_heads / kv.kv_heads, g0 = hg * plan.heads;
    w.ng = group - g0 < plan.heads ? group - g0 : plan.heads;
    w.h0 = w.head * group + g0;
    const int pos = b.kv_len[w.seq] - 1;
    w.keys = seen_keys(b, pos, pos, a.window, a.sinks);
    if (pos >= b.cap && threadIdx.x == 0) paged_flag(kv, PAGED_BAD_POSITION);
    w.lo = w.split * plan.chunk;
    if (w.split > 0 && w.lo >= w.keys.n) return false;  // the join knows
    w.hi = w.split == plan.splits - 1 || w.lo + plan.chunk > w.keys.n ? w.keys.n : w.lo + plan.chunk;
    return true;
}
// The warps' (m, l, o) of a CTA, in shared memory as [warp][G][hd], to the
// output or to the split's place in the scratch.
template <int G>
__device__ __forceinline__ void decode_store(const KvView &kv, const PagedAttnView &a, const DecodePlan &plan,
                                             const DecodeWork &w, const float *s_o, const float (*s_m)[G], const float (*s_l)[G]) {
    for (int e = threadIdx.x; e < w.ng * kv.hd; e += PD_THREADS) {
        const int g = e / kv.hd, d = e % kv.hd;
        float top = s_m[0][g];
#pragma unroll
        for (int i = 1; i < PD_WARPS; i++) top = fmaxf(top, s_m[i][g]);
        float o = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < PD_WARPS; i++) {
            const float f = exp2_approx(__fsub_rn(s_m[i][g], top));
            o = __fmaf_rn(f, s_o[(i * G + g) * kv.hd + d], o);
            sum = __fmaf_rn(f, s_l[i][g], sum);
        }
        if (plan.splits == 1) {
            a.out[(size_t)w.seq * a.ldo + (size_t)(w.h0 + g) * kv.hd + d] = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
        } else {
            const size_t at = ((size_t)w.seq * a.num_heads + w.h0 + g) * plan.splits + w.split;
            plan.part_o[at * kv.hd + d] = o;
            if (d == 0) plan.part_ml[at] = make_float2(top, sum);
        }
    }
}

// f32 pages, on the CUDA cores.
//
// LPR lanes hold one key's row (16 bytes each), so a warp reads 32/LPR rows a
// pass and a tile is 8 passes of 512 bytes whatever the head_dim.  Each lane
// dots its elements for every head; the 8 passes' partial sums are summed over
// the row's lanes by halving exchanges (4 + 2 + 1 shuffles and one more per
// doubling of LPR past 8), which leave lane i with the scores of pass i & 7.
// A warp's tiles come through its own ring of cp.async stages: no barrier of
// the CTA before its end.  Slots past the end, and pages that are not held, are
// filled with zeros and get weight zero.
template <int LPR, int G>
__global__ void __launch_bounds__(PD_THREADS, ctas_per_sm(G))
    paged_decode_kernel(KvView kv, BatchView b, PagedAttnView a, DecodePlan plan) {
    constexpr int RPP = 32 / LPR;          // rows per pass
    constexpr int TK = RPP * PD_PASSES;    // keys per tile
    constexpr int NV = 2;                  // f32 pairs per lane and row
    constexpr int E = 2 * NV;
    constexpr int ES = 4;
    constexpr int GP = (G + 1) & ~1;
    extern __shared__ __align__(128) unsigned char pd_smem[];
    __shared__ __align__(16) uint64_t s_p[PD_WARPS][TK][GP];
    __shared__ unsigned s_valid[PD_WARPS][PD_STAGES];
    __shared__ float s_m[PD_WARPS][G], s_l[PD_WARPS][G];

    pdl_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    DecodeWork work;
    if (!decode_work(kv, b, a, plan, work)) return;
    const int seq = work.seq, head = work.head, h0 = work.h0, ng = work.ng, lo = work.lo, hi = work.hi;
    const SeenKeys keys = work.keys;

    const int c = lane % LPR, rg = lane / LPR;
    const bool in_row = c * E < kv.hd;
    uint64_t q[G][NV];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const float *src = a.q + (size_t)seq * a.ldq + (size_t)(h0 + g) * kv.hd + c * E;
#pragma unroll
        for (int i = 0; i < NV; i++)
            q[g][i] = in_row && g < ng ? pack2(src[2 * i], src[2 * i + 1]) : 0ull;
    }

    const unsigned ring = smem_addr(pd_smem) + warp * (PD_STAGES * 2 * PD_TILE);
    const int ntile = (hi - lo + TK - 1) / TK;
    // element offset of key `lane` of tile t, -1 for none
    auto lookup = [&](int t) -> long long {
        const int i = lo + t * TK + lane;
        return lane < TK && t < ntile && i < hi ? key_offset(kv, b, seq, (unsigned)keys.key(i), head) : -1;
    };
    auto fill = [&](int stage, long long off) {
        const unsigned valid = __ballot_sync(0xffffffffu, off >= 0);
        if (lane == 0) s_valid[warp][stage] = valid;
        const unsigned dst = ring + stage * (2 * PD_TILE) + lane * 16;
#pragma unroll
        for (int p = 0; p < PD_PASSES; p++) {
            const long long o = __shfl_sync(0xffffffffu, off, p * RPP + rg);
            const size_t at = (o >= 0 && in_row ? (size_t)o * ES + c * 16 : 0);
            const unsigned n = o >= 0 && in_row ? 16u : 0u;
            cp_async16_zfill(dst + p * 512, reinterpret_cast<const char *>(kv.k) + at, n);
            cp_async16_zfill(dst + PD_TILE + p * 512, reinterpret_cast<const char *>(kv.v) + at, n);
        }
    };

    float m[G], l[G];
    uint64_t acc[G][NV];
#pragma unroll
    for (int g = 0; g < G; g++) {
        m[g] = NO_MAX;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) acc[g][i] = 0ull;
    }
    const float sl2 = __fmul_rn(a.scale, 1.44269504088896340736f);
    const int my_key = (lane & 7) * RPP + rg;        // the key whose scores this lane ends with
    const bool first_copy = (lane & (LPR - 1)) < 8;  // LPR / 8 lanes end with the same scores

    int t_fill = warp, stage = 0;
#pragma unroll
    for (int s = 0; s < PD_STAGES - 1; s++) {
        if (t_fill < ntile) fill(s, lookup(t_fill));
        cp_async_commit();
        t_fill += PD_WARPS;
    }
    long long off_next = lookup(t_fill);
    for (int t = warp; t < ntile; t += PD_WARPS) {
        cp_async_wait<PD_STAGES - 2>();
        __syncwarp();
        {
            const int to = stage == 0 ? PD_STAGES - 1 : stage - 1;
            if (t_fill < ntile) fill(to, off_next);
            cp_async_commit();
            t_fill += PD_WARPS;
            off_next = lookup(t_fill);
        }
        const unsigned kt = ring + stage * (2 * PD_TILE) + lane * 16, vt = kt + PD_TILE;
        float s[G][PD_PASSES];
#pragma unroll
        for (int p = 0; p < PD_PASSES; p++) {
            uint64_t x[NV];
            load_chunk(kt + p * 512, x);
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint64_t d = mul2(q[g][0], x[0]);
#pragma unroll
                for (int i = 1; i < NV; i++) d = fma2(q[g][i], x[i], d);
                float d0, d1;
                unpack2(d, d0, d1);
                s[g][p] = __fadd_rn(d0, d1);
            }
        }
        const bool up4 = lane & 4, up2 = lane & 2, up1 = lane & 1;
        float x[G];
        bool move = false;
        const bool seen = (s_valid[warp][stage] >> my_key) & 1u;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float u4[4], u2[2], u1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float give = up4 ? s[g][j] : s[g][j + 4], keep = up4 ? s[g][j + 4] : s[g][j];
                u4[j] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, 4));
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float give = up2 ? u4[j] : u4[j + 2], keep = up2 ? u4[j + 2] : u4[j];
                u2[j] = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, 2));
            }
            {
                const float give = up1 ? u2[0] : u2[1], keep = up1 ? u2[1] : u2[0];
                u1 = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, 1));
            }
#pragma unroll
            for (int o = 8; o < LPR; o <<= 1) u1 = __fadd_rn(u1, __shfl_xor_sync(0xffffffffu, u1, o));
            x[g] = seen ? __fmul_rn(u1, sl2) : -INFINITY;
            move = move || x[g] > m[g] + WeightRange<KV_F32>::rescale;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int g = 0; g < G; g++) {
                float top = x[g];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m[g]);
                const float f = exp2_approx(__fsub_rn(m[g], top));
                m[g] = top;
                l[g] = __fmul_rn(l[g], f);
                const uint64_t ff = pack2(f, f);
#pragma unroll
                for (int i = 0; i < NV; i++) acc[g][i] = mul2(acc[g][i], ff);
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float w = exp2_approx(__fsub_rn(x[g], m[g]));
            l[g] = __fadd_rn(l[g], w);
            if (first_copy) s_p[warp][my_key][g] = pack2(w, w);
        }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < PD_PASSES; p++) {
            uint64_t v[NV];
            load_chunk(vt + p * 512, v);
            const uint64_t *w = s_p[warp][p * RPP + rg];
#pragma unroll
            for (int g = 0; g < G; g++) {
                const uint64_t wg = w[g];
#pragma unroll
                for (int i = 0; i < NV; i++) acc[g][i] = fma2(wg, v[i], acc[g][i]);
            }
        }
        stage = stage == PD_STAGES - 1 ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    __syncthreads();  // every ring is free: the warps' results go there

    float *s_o = reinterpret_cast<float *>(pd_smem);  // [warp][g][hd]
#pragma unroll
    for (int g = 0; g < G; g++) {
        float sum = first_copy ? l[g] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
        if (lane == 0) s_m[warp][g] = m[g], s_l[warp][g] = sum;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float o0, o1;
            unpack2(acc[g][i], o0, o1);
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1) {
                o0 = __fadd_rn(o0, __shfl_xor_sync(0xffffffffu, o0, o));
                o1 = __fadd_rn(o1, __shfl_xor_sync(0xffffffffu, o1, o));
            }
            if (rg == 0 && in_row) {
                s_o[(warp * G + g) * kv.hd + c * E + 2 * i] = o0;
                s_o[(warp * G + g) * kv.hd + c * E + 2 * i + 1] = o1;
            }
        }
    }
    __syncthreads();
    decode_store<G>(kv, a, plan, work, s_o, s_m, s_l);
}

// f16 and bf16 pages, on the tensor cores (mma.sync m16n8k16: a warp's own,
// with fragments in registers; the 128-row tiles of tcgen05 would hold 8 rows).
//
// The 16 rows of A are up to 8 query heads in two 16-bit parts each, f16 with
// the row scaled so that its largest element is near 2^15, or the first two of
// three bf16 parts; the third has MMAs of its own.  A key's row is a column of
// B straight from shared memory (ldmatrix).  Rows h and h + 8 of the scores
// are one lane's, so it adds the parts itself, and its weights are, packed,
// the A operand of w.v: nothing crosses lanes but the row maxima, on the tiles
// where a reference moves.  Each step's w.v starts from zero and is added in
// f32: the tensor core cuts its sums.  About 500 instructions per 16 keys of
// 128 elements (f16); the same on the CUDA cores took 900: 64 sequences of 500
// to 8192 keys in f16 238 us there and 194 here, 64 of 2049 (9 / 3 heads of 64)
// 28.7 and 25.6.  bf16 pays for its third part: 230 and 223, 28.1 and 28.5; 128
// windows of 1028 keys 112.5 and 114.5, one sequence of 8192 18.5 and 19.1.  It is
// bound by memory (5 to 5.9 TB/s of pages scattered over the pool).
__device__ __forceinline__ void ldsm4(unsigned a, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(unsigned a, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
template <int TYPE>
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
    if constexpr (TYPE == KV_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
template <int TYPE>
__device__ __forceinline__ void mma16816_zero(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                              unsigned b1) {
    if constexpr (TYPE == KV_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

template <int TYPE, int LPR>
__global__ void __launch_bounds__(PD_THREADS, 3)
    paged_decode_mma_kernel(KvView kv, BatchView b, PagedAttnView a, DecodePlan plan) {
    constexpr int G = 8;
    constexpr int RPP = 32 / LPR, TK = RPP * PD_PASSES;  // keys per tile: 16 or 32
    constexpr int ROW = LPR * 16;                        // bytes of a key's row
    constexpr int KS = LPR / 2;                          // 16-element steps of a row
    constexpr int NQ = TYPE == KV_F16 ? 2 : 3;
    using Range = WeightRange<TYPE>;
    // the products of the first and of the second part
    auto sum2 = [](float p0, float p1) {
        return TYPE == KV_F16 ? __fmaf_rn(p1, F16_PART2_INV, p0) : __fadd_rn(p0, p1);
    };
    extern __shared__ __align__(128) unsigned char pd_smem[];
    __shared__ unsigned s_valid[PD_WARPS][PD_STAGES];
    __shared__ float s_m[PD_WARPS][G], s_l[PD_WARPS][G];

    pdl_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    DecodeWork work;
    if (!decode_work(kv, b, a, plan, work)) return;
    const int seq = work.seq, head = work.head, lo = work.lo, hi = work.hi;
    const SeenKeys keys = work.keys;

    // this lane's head and element pairs: 16 ks + 2 (lane & 3) + {0, 1} and 8 on
    const int g = lane >> 2, e0 = (lane & 3) * 2;
    float sl2 = __fmul_rn(a.scale, 1.44269504088896340736f);
    unsigned qa[KS][2][NQ];  // [step][first or second half of it][part]
    {
        const float *src = a.q + (size_t)seq * a.ldq + (size_t)(work.h0 + (g < work.ng ? g : 0)) * kv.hd;
        float f[KS][4];
        unsigned top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = ks * 16 + e0 + (i & 1) + (i >> 1) * 8;
                f[ks][i] = d < kv.hd && g < work.ng ? src[d] : 0.f;
                top = max(top, __float_as_uint(fabsf(f[ks][i])));
            }
        float up = 1.0f;
        if constexpr (TYPE == KV_F16) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int e = 141 - (int)(top >> 23);  // 2^14 <= top 2^e < 2^15
            e = top == 0 || top >= 0x7f800000u ? 0 : e > 120 ? 120 : e;
            up = __uint_as_float((unsigned)(127 + e) << 23);
            sl2 = __fmul_rn(sl2, __uint_as_float((unsigned)(127 - e) << 23));
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                split2<TYPE, NQ>(__fmul_rn(f[ks][2 * i], up), __fmul_rn(f[ks][2 * i + 1], up), qa[ks][i]);
    }

    const unsigned ring = smem_addr(pd_smem) + warp * (PD_STAGES * 2 * PD_TILE);
    const int ntile = (hi - lo + TK - 1) / TK;
    const int c = lane % LPR, rg = lane / LPR;
    const bool in_row = c * 8 < kv.hd;
    auto lookup = [&](int t) -> long long {  // byte offset of key `lane` of tile t, -1 for none
        const int i = lo + t * TK + lane;
        const long long o = lane < TK && t < ntile && i < hi ? key_offset(kv, b, seq, (unsigned)keys.key(i), head) : -1;
        return o < 0 ? -1 : 2 * o;
    };
    // 16-byte chunk c of row r is at chunk c ^ (r & 7): eight rows' chunks of
    // one matrix lie in different banks
    const char *const k_at = reinterpret_cast<const char *>(kv.k) + (in_row ? c * 16 : 0);
    const char *const v_at = reinterpret_cast<const char *>(kv.v) + (in_row ? c * 16 : 0);
    auto fill = [&](int stage, long long off) {
        const unsigned valid = __ballot_sync(0xffffffffu, off >= 0);
        if (lane == 0) s_valid[warp][stage] = valid;
        if (off < 0) off = 0;
        const unsigned mine = in_row ? valid : 0u;
        const unsigned dst = ring + stage * (2 * PD_TILE);
#pragma unroll
        for (int p = 0; p < PD_PASSES; p++) {
            const int r = p * RPP + rg;
            const long long o = __shfl_sync(0xffffffffu, off, r);
            const unsigned n = (mine >> r) << 4 & 16u, to = dst + r * ROW + ((c ^ (r & 7)) << 4);
            cp_async16_zfill(to, k_at + o, n);
            cp_async16_zfill(to + PD_TILE, v_at + o, n);
        }
    };

    float m = NO_MAX, l = 0.f;
    float acc[LPR][2];  // elements 8 t + e0 + {0, 1} of the head's output
#pragma unroll
    for (int t = 0; t < LPR; t++) acc[t][0] = acc[t][1] = 0.f;

    int t_fill = warp, stage = 0;
#pragma unroll
    for (int s = 0; s < PD_STAGES - 1; s++) {
        if (t_fill < ntile) fill(s, lookup(t_fill));
        cp_async_commit();
        t_fill += PD_WARPS;
    }
    long long off_next = lookup(t_fill);
    const int lr = lane & 7, lm = lane >> 3;  // row and matrix this lane addresses
    for (int t = warp; t < ntile; t += PD_WARPS) {
        cp_async_wait<PD_STAGES - 2>();
        __syncwarp();
        {
            const int to = stage == 0 ? PD_STAGES - 1 : stage - 1;
            if (t_fill < ntile) fill(to, off_next);
            cp_async_commit();
            t_fill += PD_WARPS;
            off_next = lookup(t_fill);
        }
        const unsigned kt = ring + stage * (2 * PD_TILE), vt = kt + PD_TILE;
        const unsigned valid = s_valid[warp][stage];
        float x[TK / 8][2];
        bool move = false;
#pragma unroll
        for (int n = 0; n < TK / 8; n++) {  // eight keys
            float s01[4], s2[4];
#pragma unroll
            for (int k2 = 0; k2 < KS / 2; k2++) {
                unsigned kb[4];
                ldsm4(kt + (n * 8 + lr) * ROW + (((k2 * 4 + lm) ^ lr) << 4), kb);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const unsigned(&q)[2][NQ] = qa[k2 * 2 + i];
                    if (k2 + i == 0) {
                        mma16816_zero<TYPE>(s01, q[0][0], q[0][1], q[1][0], q[1][1], kb[0], kb[1]);
                        if constexpr (NQ == 3) mma16816_zero<TYPE>(s2, q[0][2], 0u, q[1][2], 0u, kb[0], kb[1]);
                    } else {
                        mma16816<TYPE>(s01, q[0][0], q[0][1], q[1][0], q[1][1], kb[2 * i], kb[2 * i + 1]);
                        if constexpr (NQ == 3) mma16816<TYPE>(s2, q[0][2], 0u, q[1][2], 0u, kb[2 * i], kb[2 * i + 1]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float s = sum2(s01[i], s01[2 + i]);
                if constexpr (NQ == 3) s = __fadd_rn(s, s2[i]);
                x[n][i] = (valid >> (n * 8 + e0 + i)) & 1u ? __fmul_rn(s, sl2) : -INFINITY;
                move = move || x[n][i] > m + Range::rescale;
            }
        }
        if (__any_sync(0xffffffffu, move)) {
            float top = x[0][0];
#pragma unroll
            for (int n = 0; n < TK / 8; n++) top = fmaxf(top, fmaxf(x[n][0], x[n][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(__fsub_rn(top, Range::margin), m);
            const float f = exp2_approx(__fsub_rn(m, top));
            m = top;
            l = __fmul_rn(l, f);
#pragma unroll
            for (int d = 0; d < LPR; d++) acc[d][0] = __fmul_rn(acc[d][0], f), acc[d][1] = __fmul_rn(acc[d][1], f);
        }
        unsigned w[TK / 8][NQ];
#pragma unroll
        for (int n = 0; n < TK / 8; n++) {
            const float w0 = exp2_approx(__fsub_rn(x[n][0], m)), w1 = exp2_approx(__fsub_rn(x[n][1], m));
            l = __fadd_rn(l, __fadd_rn(w0, w1));
            split2_weights<TYPE, NQ>(w0, w1, w[n]);
        }
#pragma unroll
        for (int d2 = 0; d2 < LPR / 2; d2++) {  // sixteen elements
            float o0[4], o1[4];
#pragma unroll
            for (int u = 0; u < TK / 16; u++) {
                unsigned vb[4];
                ldsm4_t(vt + (u * 16 + (lm & 1) * 8 + lr) * ROW + (((d2 * 2 + (lm >> 1)) ^ lr) << 4), vb);
                auto add = [&](bool zero, unsigned a0, unsigned a1, unsigned a2, unsigned a3) {
                    if (zero) {
                        mma16816_zero<TYPE>(o0, a0, a1, a2, a3, vb[0], vb[1]);
                        mma16816_zero<TYPE>(o1, a0, a1, a2, a3, vb[2], vb[3]);
                    } else {
                        mma16816<TYPE>(o0, a0, a1, a2, a3, vb[0], vb[1]);
                        mma16816<TYPE>(o1, a0, a1, a2, a3, vb[2], vb[3]);
                    }
                };
                if constexpr (NQ == 3) add(u == 0, w[2 * u][2], 0u, w[2 * u + 1][2], 0u);
                add(u == 0 && NQ == 2, w[2 * u][0], w[2 * u][1], w[2 * u + 1][0], w[2 * u + 1][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                acc[2 * d2][i] = __fadd_rn(acc[2 * d2][i], sum2(o0[i], o0[2 + i]));
                acc[2 * d2 + 1][i] = __fadd_rn(acc[2 * d2 + 1][i], sum2(o1[i], o1[2 + i]));
            }
        }
        __syncwarp();  // the stage is filled again at the next turn
        stage = stage == PD_STAGES - 1 ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    __syncthreads();  // every ring is free: the warps' results go there

    float *s_o = reinterpret_cast<float *>(pd_smem);  // [warp][head][hd]
    l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 1));
    l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 2));
    if ((lane & 3) == 0) s_m[warp][g] = m, s_l[warp][g] = l;
#pragma unroll
    for (int d = 0; d < LPR; d++)
        if (d * 8 < kv.hd) {
            s_o[(warp * G + g) * kv.hd + d * 8 + e0] = acc[d][0];
            s_o[(warp * G + g) * kv.hd + d * 8 + e0 + 1] = acc[d][1];
        }
    bool finite = fabsf(l) < INFINITY;
#pragma unroll
    for (int d = 0; d < LPR; d++) finite = finite && fabsf(acc[d][0]) < INFINITY && fabsf(acc[d][1]) < INFINITY;
    if (__syncthreads_or(!finite && g < work.ng)) {
        // warp 0's place gets each head's whole result, the others' nothing
        for (int h = warp; h < work.ng; h += PD_WARPS) {
            const RowState st = attend_row<TYPE>(kv, b, seq, head, a.q + (size_t)seq * a.ldq + (size_t)(work.h0 + h) * kv.hd,
                                                 __fmul_rn(a.scale, 1.44269504088896340736f), keys, lo, hi, 0, 0, 0x7fffffff);
            for (int i = 0; i < PD_WARPS; i++) {
#pragma unroll
                for (int c4 = 0; c4 < 4; c4++)
                    if (lane + 32 * c4 < kv.hd) s_o[(i * G + h) * kv.hd + lane + 32 * c4] = i == 0 ? st.acc[c4] : 0.f;
                if (lane == 0) s_m[i][h] = i == 0 ? st.m : NO_MAX, s_l[i][h] = i == 0 ? st.l : 0.f;
            }
        }
        __syncthreads();
    }
    decode_store<G>(kv, a, plan, work, s_o, s_m, s_l);
}

// Joins the splits of one (row, query head): warp w takes splits w, w + 4, ..
// (four loads in flight), a lane four elements of head_dim, and the warps'
// sums meet in shared memory.
constexpr int PJ_WARPS = 4;
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_join_kernel(KvView kv, BatchView b, PagedAttnView a, const float2 *part_ml,
                                                                       const float *part_o, int chunk, int splits) {
    __shared__ float4 s_o[PJ_WARPS][32];
    __shared__ float s_l[PJ_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t item = blockIdx.x;
    const int row = (int)(item / (unsigned)a.num_heads), h = (int)(item % (unsigned)a.num_heads);
    int live = splits;
    bool owned = true;
    if (chunk > 0) {
        const int pos = b.kv_len[row] - 1;  // not written by the kernel waited for
        const SeenKeys keys = seen_keys(b, pos, pos, a.window, a.sinks);
        live = (int)(((unsigned)keys.n + (unsigned)chunk - 1u) / (unsigned)chunk);
        live = live < 1 ? 1 : live > splits ? splits : live;
    } else {
        owned = row >= b.row_start[0] && row < b.row_start[b.num_seqs];
    }
    // every CTA waits, those without work too: else a join of rows that are no
    // sequence's would end, and let its own successor start, before they are zeroed
    pdl_wait();
    if (!owned) return;
    const float2 *ml = part_ml + item * splits;
    const float *po = part_o + item * splits * (uint64_t)kv.hd + 4 * lane;
    const bool mine = 4 * lane < kv.hd;
    float top = NO_MAX;
    for (int s = lane; s < live; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = warp; s0 < live; s0 += 4 * PJ_WARPS) {
        float2 x[4];
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int s = s0 + u * PJ_WARPS;
            x[u] = s < live ? ml[s] : make_float2(NO_MAX, 0.f);
            v[u] = s < live && mine ? *reinterpret_cast<const float4 *>(po + (size_t)s * kv.hd) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float f = exp2_approx(__fsub_rn(x[u].x, top));
            sum = __fmaf_rn(f, x[u].y, sum);
            acc.x = __fmaf_rn(f, v[u].x, acc.x);
            acc.y = __fmaf_rn(f, v[u].y, acc.y);
            acc.z = __fmaf_rn(f, v[u].z, acc.z);
            acc.w = __fmaf_rn(f, v[u].w, acc.w);
        }
    }
    s_o[warp][lane] = acc;
    if (lane == 0) s_l[warp] = sum;
    __syncthreads();
    const float total = __fadd_rn(__fadd_rn(s_l[0], s_l[1]), __fadd_rn(s_l[2], s_l[3]));
    const float *f = reinterpret_cast<const float *>(s_o);
    const int d = threadIdx.x;
    if (d < kv.hd) {
        const float o = __fadd_rn(__fadd_rn(f[d], f[128 + d]), __fadd_rn(f[256 + d], f[384 + d]));
        a.out[(size_t)row * a.ldo + (size_t)h * kv.hd + d] = total == 0.f ? 0.f : __fdiv_rn(o, total);
    }
}

constexpr size_t PD_SMEM = (size_t)PD_WARPS * PD_STAGES * 2 * PD_TILE;

template <typename K>
void go(K *kernel, SmemOptIn &opt, const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan,
        cudaStream_t s) {
    const unsigned grid = (unsigned)((uint64_t)b.num_seqs * kv.kv_heads * plan.head_groups * plan.splits);
    opt(kernel, (int)PD_SMEM);
    launch_kernel(kernel, dim3(grid), dim3(PD_THREADS), PD_SMEM, s, false, kv, b, a, plan);
}
template <int TYPE, int LPR>
void go_mma(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan, cudaStream_t s) {
    static SmemOptIn opt;
    go(paged_decode_mma_kernel<TYPE, LPR>, opt, kv, b, a, plan, s);
}
template <int LPR, int G>
void go_fma(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan, cudaStream_t s) {
    static SmemOptIn opt;
    go(paged_decode_kernel<LPR, G>, opt, kv, b, a, plan, s);
}
template <int LPR>
void go_heads(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan, cudaStream_t s) {
    switch (plan.heads) {
        case 1: go_fma<LPR, 1>(kv, b, a, plan, s); break;
        case 2: go_fma<LPR, 2>(kv, b, a, plan, s); break;
        case 3: go_fma<LPR, 3>(kv, b, a, plan, s); break;
        case 4: go_fma<LPR, 4>(kv, b, a, plan, s); break;
        case 6: go_fma<LPR, 6>(kv, b, a, plan, s); break;
        default: go_fma<LPR, 8>(kv, b, a, plan, s); break;
    }
}

}  // namespace

DecodePlan plan_paged_decode(const KvView &kv, const BatchView &b, const PagedAttnView &a, uint32_t max_kv_len) {
    DecodePlan p{};
    const int group = a.num_heads / kv.kv_heads;
    // query heads of a KV head in one CTA: up to 8 share each key they read
    p.head_groups = (group + 7) / 8;
    const int g = (group + p.head_groups - 1) / p.head_groups;
    p.heads = kv.type != KV_F32 ? 8 : g == 5 ? 6 : g == 7 ? 8 : g;
    p.head_groups = (group + p.heads - 1) / p.heads;
    uint64_t most = max_kv_len;
    if (a.window) most = std::min<uint64_t>(most, (uint64_t)a.window + a.sinks);
    most = std::max<uint64_t>(most, 1);
    const uint64_t units = std::max<uint64_t>((uint64_t)b.num_seqs * kv.kv_heads * p.head_groups, 1);
    // Of 1 to 64 splits the cheapest by this count, in bytes of an SM's share of
    // the memory's rate: the keys of the SM with the most CTAs, a start and an
    // end per wave of CTAs (about 5 us), and the join's launch (about 4 us).
    // Where two are within 3 % the fewer splits win.  Measured, with cold
    // pages: 64 x 2049 f32, 192 units: 1, 2, 3, 4 splits 54, 50, 59, 54 us; one
    // sequence of 8192 f16, 8 units: 8, 16, 24, 32, 48 splits 28, 21.5, 23.5,
    // 21.5, 23.6 us; 64 sequences of 500 to 8192 bf16, 512 units: 1, 2, 4, 8, 12
    // splits 289, 257, 226, 228, 241 us; 128 windows of 1028 keys f16, 1024
    // units: 1, 2, 3 splits 115, 120, 124 us.
    constexpr uint64_t SMS = 148, WAVE = 215 << 10, JOIN = 170 << 10;
    const uint64_t slots = SMS * (uint64_t)(kv.type == KV_F32 ? ctas_per_sm(p.heads) : 3);
    const uint64_t key_bytes = 2ull * kv.hd * (kv.type == KV_F32 ? 4 : 2);
    uint64_t best = UINT64_MAX;
    // lengths below the bound may be unlike: with at most 1 MB a CTA the last end together
    const uint64_t fewest = std::min<uint64_t>(64, std::max<uint64_t>(1, (most * key_bytes) >> 20));
    for (uint64_t s = fewest; s <= 64; s++) {
        const uint64_t chunk = ((most + s - 1) / s + 15) / 16 * 16;
        const uint64_t ctas = units * s;
        // (past eight waves the count seldom wins, and the scratch has its bound)
        if (s > fewest && (chunk < 64 || ctas > 8 * slots)) break;
        const uint64_t waves = (ctas + slots - 1) / slots, deep = (ctas + SMS - 1) / SMS;
        const uint64_t cost = deep * chunk * key_bytes + waves * WAVE + (s > 1 ? JOIN : 0);
        if (best != UINT64_MAX && cost + cost / 32 >= best) continue;
        best = cost;
        p.chunk = (int)std::min<uint64_t>(chunk, INT32_MAX);
        p.splits = (int)((most + chunk - 1) / chunk);
    }
    const uint64_t rows = (uint64_t)b.num_rows * a.num_heads, parts = p.splits > 1 ? rows * p.splits : 0;
    p.ml_bytes = parts_ml_bytes(parts);
    // The bound for every call of as many rows and keys or fewer, which may be
    // split more: as often as `fewest` says, or with chunks of 64 keys (so that
    // the splits are fewer than most / 48) and at most 8 x slots CTAs.
    const uint64_t more = std::min<uint64_t>(64, most / 48);
    uint64_t bound = fewest > 1 ? rows * fewest : 0;
    if (more > 1) bound = std::max(bound, std::min(rows * more, 8 * slots * (uint64_t)p.heads));
    p.scratch_bytes = parts_bytes(std::max(parts, bound), kv.hd);
    return p;
}

void launch_paged_decode(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan,
                         cudaStream_t s) {
    if (kv.type == KV_F32)
        kv.hd <= 64 ? go_heads<16>(kv, b, a, plan, s) : go_heads<32>(kv, b, a, plan, s);
    else if (kv.type == KV_F16)
        kv.hd <= 64 ? go_mma<KV_F16, 8>(kv, b, a, plan, s) : go_mma<KV_F16, 16>(kv, b, a, plan, s);
    else
        kv.hd <= 64 ? go_mma<KV_BF16, 8>(kv, b, a, plan, s) : go_mma<KV_BF16, 16>(kv, b, a, plan, s);
    if (plan.splits > 1) launch_paged_join(kv, b, a, plan.part_ml, plan.part_o, plan.chunk, plan.splits, s);
}

void launch_paged_join(const KvView &kv, const BatchView &b, const PagedAttnView &a, const float2 *part_ml,
                       const float *part_o, int chunk, int splits, cudaStream_t s) {
    const uint64_t items = (uint64_t)b.num_rows * a.num_heads;
    launch_kernel(paged_join_kernel, dim3((unsigned)items), dim3(PJ_WARPS * 32), 0, s, true, kv, b, a, part_ml, part_o,
                  chunk, splits);
}

}  // namespace slm
