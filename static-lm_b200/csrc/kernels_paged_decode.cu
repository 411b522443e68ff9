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
constexpr float PD_NO_MAX = -3.0e38f;      // below every finite score
constexpr float PD_RESCALE = 8.0f;         // the reference moves when a score passes it by 2^8

// CTAs of g query heads that an SM holds: by shared memory, and by registers.
__host__ __device__ constexpr int ctas_per_sm(int g) { return g <= 4 ? 3 : 2; }

__device__ __forceinline__ void cp_async16_zfill(unsigned dst, const void *src, unsigned bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}

// The 16 bytes of one lane as f32 pairs.
template <int TYPE>
struct Chunk;
template <>
struct Chunk<KV_F32> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void get(unsigned a, uint64_t (&x)[2]) {
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(x[0]), "=l"(x[1]) : "r"(a));
    }
};
template <>
struct Chunk<KV_F16> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(unsigned a, uint64_t (&x)[4]) {
        unsigned w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[i] = pack2(f.x, f.y);
        }
    }
};
template <>
struct Chunk<KV_BF16> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(unsigned a, uint64_t (&x)[4]) {
        unsigned w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
};

// Work of one CTA: keys [split*chunk, ..) of the list of keys that the row of
// sequence `seq` sees (the last split takes what is left), KV head `head`,
// `g` query heads from h0 on.
//
// LPR lanes hold one key's row (16 bytes each), so a warp reads 32/LPR rows a
// pass and a tile is 8 passes of 512 bytes whatever the type and head_dim.
// Each lane dots its elements for every head; the 8 passes' partial sums are
// summed over the row's lanes by halving exchanges (4 + 2 + 1 shuffles and
// one more per doubling of LPR past 8), which leave lane i with the scores of
// pass i & 7.  A warp's tiles come through its own ring of cp.async stages:
// no barrier of the CTA before the join.  Slots past the end, and pages that
// are not held, are filled with zeros and get weight zero.
template <int TYPE, int LPR, int G>
__global__ void __launch_bounds__(PD_THREADS, ctas_per_sm(G))
    paged_decode_kernel(KvView kv, BatchView b, PagedAttnView a, DecodePlan plan) {
    constexpr int RPP = 32 / LPR;          // rows per pass
    constexpr int TK = RPP * PD_PASSES;    // keys per tile
    constexpr int NV = Chunk<TYPE>::N;     // f32 pairs per lane and row
    constexpr int E = 2 * NV;
    constexpr int ES = TYPE == KV_F32 ? 4 : 2;
    constexpr int GP = (G + 1) & ~1;
    extern __shared__ __align__(128) unsigned char pd_smem[];
    __shared__ __align__(16) uint64_t s_p[PD_WARPS][TK][GP];
    __shared__ unsigned s_valid[PD_WARPS][PD_STAGES];
    __shared__ float s_m[PD_WARPS][G], s_l[PD_WARPS][G];

    pdl_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int split = blockIdx.x % plan.splits;
    int unit = blockIdx.x / plan.splits;
    const int hg = unit % plan.head_groups;
    unit /= plan.head_groups;
    const int head = unit % kv.kv_heads, seq = unit / kv.kv_heads;
    const int group = a.num_heads / kv.kv_heads;
    const int g0 = hg * G, ng = group - g0 < G ? group - g0 : G;
    const int h0 = head * group + g0;

    const int pos = b.kv_len[seq] - 1;
    const SeenKeys keys = seen_keys(pos, pos, a.window, a.sinks);
    const int lo = split * plan.chunk;
    if (split > 0 && lo >= keys.n) return;  // the join knows
    const int hi = split == plan.splits - 1 || lo + plan.chunk > keys.n ? keys.n : lo + plan.chunk;

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
        m[g] = PD_NO_MAX;
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
            Chunk<TYPE>::get(kt + p * 512, x);
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
            move = move || x[g] > m[g] + PD_RESCALE;
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
            Chunk<TYPE>::get(vt + p * 512, v);
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
    for (int e = threadIdx.x; e < ng * kv.hd; e += PD_THREADS) {
        const int g = e / kv.hd, d = e % kv.hd;
        float top = s_m[0][g];
#pragma unroll
        for (int w = 1; w < PD_WARPS; w++) top = fmaxf(top, s_m[w][g]);
        float o = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < PD_WARPS; w++) {
            const float f = exp2_approx(__fsub_rn(s_m[w][g], top));
            o = __fmaf_rn(f, s_o[(w * G + g) * kv.hd + d], o);
            sum = __fmaf_rn(f, s_l[w][g], sum);
        }
        if (plan.splits == 1) {
            a.out[(size_t)seq * a.ldo + (size_t)(h0 + g) * kv.hd + d] = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
        } else {
            const size_t at = ((size_t)seq * a.num_heads + h0 + g) * plan.splits + split;
            plan.part_o[at * kv.hd + d] = o;
            if (d == 0) plan.part_ml[at] = make_float2(top, sum);
        }
    }
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
    if (chunk > 0) {
        const int pos = b.kv_len[row] - 1;  // not written by the kernel waited for
        const SeenKeys keys = seen_keys(pos, pos, a.window, a.sinks);
        live = (keys.n + chunk - 1) / chunk;
        live = live < 1 ? 1 : live > splits ? splits : live;
    } else if (row >= b.row_start[b.num_seqs]) {
        return;  // no sequence's: zeroed already
    }
    pdl_wait();
    const float2 *ml = part_ml + item * splits;
    const float *po = part_o + item * splits * (uint64_t)kv.hd + 4 * lane;
    const bool mine = 4 * lane < kv.hd;
    float top = PD_NO_MAX;
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
            x[u] = s < live ? ml[s] : make_float2(PD_NO_MAX, 0.f);
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

template <int TYPE, int LPR, int G>
void go(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan, cudaStream_t s) {
    const unsigned grid = (unsigned)((uint64_t)b.num_seqs * kv.kv_heads * plan.head_groups * plan.splits);
    static SmemOptIn opt;
    opt(paged_decode_kernel<TYPE, LPR, G>, (int)PD_SMEM);
    launch_kernel(paged_decode_kernel<TYPE, LPR, G>, dim3(grid), dim3(PD_THREADS), PD_SMEM, s, false, kv, b, a, plan);
}

template <typename F>
void for_heads(int g, F f) {
    switch (g) {
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 3: f(std::integral_constant<int, 3>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        case 6: f(std::integral_constant<int, 6>{}); break;
        default: f(std::integral_constant<int, 8>{}); break;
    }
}

// f(type, lanes per row): rows of up to 64 or up to 128 elements
template <typename F>
void for_rows(int type, int hd, F f) {
    if (type == KV_F32) {
        if (hd <= 64)
            f(std::integral_constant<int, KV_F32>{}, std::integral_constant<int, 16>{});
        else
            f(std::integral_constant<int, KV_F32>{}, std::integral_constant<int, 32>{});
    } else if (type == KV_F16) {
        if (hd <= 64)
            f(std::integral_constant<int, KV_F16>{}, std::integral_constant<int, 8>{});
        else
            f(std::integral_constant<int, KV_F16>{}, std::integral_constant<int, 16>{});
    } else {
        if (hd <= 64)
            f(std::integral_constant<int, KV_BF16>{}, std::integral_constant<int, 8>{});
        else
            f(std::integral_constant<int, KV_BF16>{}, std::integral_constant<int, 16>{});
    }
}

}  // namespace

DecodePlan plan_paged_decode(const KvView &kv, const BatchView &b, const PagedAttnView &a, uint32_t max_kv_len) {
    DecodePlan p{};
    const int group = a.num_heads / kv.kv_heads;
    // query heads of a KV head in one CTA: up to 8 share each key they read
    p.head_groups = (group + 7) / 8;
    const int g = (group + p.head_groups - 1) / p.head_groups;
    p.heads = g == 5 ? 6 : g == 7 ? 8 : g;
    p.head_groups = (group + p.heads - 1) / p.heads;
    uint64_t most = max_kv_len;
    if (a.window) most = std::min<uint64_t>(most, (uint64_t)a.window + a.sinks);
    most = std::max<uint64_t>(most, 1);
    const uint64_t units = std::max<uint64_t>((uint64_t)b.num_seqs * kv.kv_heads * p.head_groups, 1);
    // A CTA costs its keys' bytes and about 150 KB more (its first look-ups and
    // copies, its warps' join); the CTAs run in waves over the SMs; the second
    // launch costs about 75 KB.  Of 1 to 64 splits the cheapest by that count.
    // Measured (best of a sweep in brackets): 64 x 2049 f32, 192 units: 2
    // splits, 50 us (1: 54, 4: 54); one sequence of 8192, 8 units: 24 to 37
    // alike; 64 ragged to 8192, 512 units: 6, 218 us (8: 216, 4: 224, 1: 315);
    // 128 windows of 1028, 1024 units: 1, 121 us (2: 126).
    const uint64_t slots = 148 * (uint64_t)ctas_per_sm(p.heads);
    const uint64_t key_bytes = 2ull * kv.hd * (kv.type == KV_F32 ? 4 : 2);
    uint64_t best = UINT64_MAX;
    for (uint64_t s = 1; s <= 64; s++) {
        uint64_t chunk = ((most + s - 1) / s + 15) / 16 * 16;
        if (s > 1 && chunk < 64) break;
        const uint64_t waves = (units * s + slots - 1) / slots;
        const uint64_t cost = waves * (chunk * key_bytes + (150 << 10)) + (s > 1 ? 75 << 10 : 0);
        if (cost >= best) continue;
        best = cost;
        p.chunk = (int)std::min<uint64_t>(chunk, INT32_MAX);
        p.splits = (int)((most + chunk - 1) / chunk);
    }
    const uint64_t parts = (uint64_t)b.num_rows * a.num_heads * p.splits;
    p.ml_bytes = p.splits > 1 ? (parts * sizeof(float2) + 15) / 16 * 16 : 0;
    p.scratch_bytes = p.splits > 1 ? p.ml_bytes + parts * kv.hd * sizeof(float) : 0;
    return p;
}

void launch_paged_decode(const KvView &kv, const BatchView &b, const PagedAttnView &a, const DecodePlan &plan,
                         cudaStream_t s) {
    for_rows(kv.type, kv.hd, [&](auto type, auto lpr) {
        for_heads(plan.heads, [&](auto g) { go<decltype(type)::value, decltype(lpr)::value, decltype(g)::value>(kv, b, a, plan, s); });
    });
    if (plan.splits > 1) launch_paged_join(kv, b, a, plan.part_ml, plan.part_o, plan.chunk, plan.splits, s);
}

void launch_paged_join(const KvView &kv, const BatchView &b, const PagedAttnView &a, const float2 *part_ml,
                       const float *part_o, int chunk, int splits, cudaStream_t s) {
    const uint64_t items = (uint64_t)b.num_rows * a.num_heads;
    launch_kernel(paged_join_kernel, dim3((unsigned)items), dim3(PJ_WARPS * 32), 0, s, true, kv, b, a, part_ml, part_o,
                  chunk, splits);
}

}  // namespace slm
