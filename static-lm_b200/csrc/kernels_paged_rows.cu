// kernels_paged_rows.cu -- attention of several new rows per sequence (a
// prompt, or a chunk behind an earlier context) over the paged cache, on the
// tcgen05 tensor cores at f32 accuracy.
//
// The tensor cores multiply 16-bit operands exactly and add in f32, so an f32
// operand is written as a sum of 16-bit parts and the products of the parts
// are added up:
//   f16 pages:  q 2^e = q0 + q1 (e per row, so that the row's largest element
//               is near 2^15: 22 bits of it survive), w = w0 + w1 for the
//               softmax weights w <= 2^8; 2 products each for q.k and w.v.
//   bf16 pages: three bf16 parts of q and w (24 bits), 3 products each.
//   f32 pages:  three bf16 parts of q, w, k and v; the 6 products whose size
//               is above 2^-24 of the leading one.
//
// A CTA takes one (sequence, KV head) and a run of its rows, the query heads
// of the KV head side by side (row = token * group + head in group), so every
// key read serves all of them.  Two streams of work keep the tensor core busy
// while the other's softmax runs: with f16 pages two tiles of 128 rows over
// the same keys, else one tile of 128 rows over the even and the odd key tiles
// (their sums are joined at the end).  Warps 0-3 and 4-7 run the streams'
// softmax, a row per thread; warp 8 issues the MMAs; warps 9-11 bring keys and
// values from the pages into a ring of shared-memory slots.
#include "async.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace slm {

namespace {

constexpr int PR_THREADS = 384;
constexpr int PR_PRODUCERS = 96;
constexpr float PR_NO_MAX = -3.0e38f;
constexpr float PR_RESCALE = 8.0f;
constexpr unsigned PR_TMEM_COLS = 512;

template <int TYPE, int HDP>
struct RowsCfg {
    static constexpr bool F16 = TYPE == KV_F16;
    static constexpr int T = F16 ? 2 : 1;        // row tiles per CTA
    static constexpr int KT = F16 ? 128 : 64;    // keys per tile
    static constexpr int NQ = F16 ? 2 : 3;       // parts of q and of the weights
    static constexpr int NC = TYPE == KV_F32 ? 3 : 1;  // parts of k and v
    static constexpr int RT = T * 128;
    static constexpr int PART = KT * HDP * 2;    // bytes of one part of a key tile
    static constexpr int SLOT = PART * NC;
    static constexpr int QPART = 128 * HDP * 2;
    static constexpr int QBYTES = T * NQ * QPART;
    static constexpr int NSLOT = F16 ? (HDP == 128 ? 3 : 6) : TYPE == KV_BF16 ? (HDP == 128 ? 6 : 8) : (HDP == 128 ? 2 : 4);
    static constexpr int SP = F16 ? 128 : 96;    // TMEM columns of scores / weights
    static constexpr int STREAM = SP + HDP;      // TMEM columns of a stream
    static constexpr int BIG = QBYTES + NSLOT * SLOT;
    // at least 120 KB: one CTA per SM, whose TMEM it takes whole
    static constexpr int SMEM = (BIG > 120 * 1024 ? BIG : 120 * 1024) + 3072;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(2 * STREAM <= (int)PR_TMEM_COLS, "TMEM");
    static_assert(QBYTES >= 128 * HDP * 4, "the odd stream's sums fit the q tiles");
};

// The small shared data, after the tiles.
struct RowsShared {
    uint64_t full[8], empty[8], s_full[2], p_full[2], o_full[2], q_full, drain;
    long long off[128];       // element offsets of the keys of the newest tiles
    float ml[2][128];         // the odd stream's maxima and sums
    unsigned valid[8][4];     // held keys of the newest 8 tiles
    unsigned taddr;
    int abort;
    // the CTA's work
    int seq, row0, rows, tile, found;  // row0: first activation row of the sequence
};
static_assert(sizeof(RowsShared) <= 3072, "small shared data");

// ---- 16-bit operands
// Byte offset of 16-byte chunk c (8 elements) of row r in the 128-byte
// swizzled layout of R rows: panels of 64 elements, R rows of 128 B each.
__device__ __forceinline__ unsigned sw16_off(int r, int c, int R) {
    return (unsigned)((c >> 3) * R * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// Descriptor of an operand whose rows run along K of the product (values: a
// row per key, head_dim contiguous): 64-element panels `panel` bytes apart
// (leading offset), 8-row groups 1024 B apart (stride offset), 128-byte swizzle.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(unsigned saddr, unsigned panel) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)((panel >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}
// Instruction descriptor of kind::f16: f32 accumulator, f16 (0) or bf16 (1)
// operands, A along K, B along K or (mn) along N.
__device__ __forceinline__ unsigned umma_idesc_f16(bool bf16, int M, int N, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24);
}
// D[128 x N] (+)= A[128 x 16] B[N x 16]^T; A in shared memory or in TMEM.
__device__ __forceinline__ void tc_mma_f16(unsigned d, uint64_t adesc, uint64_t bdesc, unsigned idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"((unsigned)acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ta(unsigned d, unsigned a, uint64_t bdesc, unsigned idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"((unsigned)acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}

// ---- TMEM <-> registers, 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(unsigned taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
// keeps uses of v after an earlier wait
__device__ __forceinline__ void pin32(float *v) {
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                   "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                   "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                   "+f"(v[29]), "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ __forceinline__ void tmem_st16(unsigned taddr, const unsigned *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 8 columns of this thread's lane times f.
__device__ __forceinline__ void tmem_scale8(unsigned taddr, float f) {
    float v[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr)
                 : "memory");
    tmem_wait_ld();
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])::"memory");
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __fmul_rn(v[i], f);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "f"(v[0]),
                 "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A bounded wait; false once any wait of the CTA gave up.
__device__ __forceinline__ bool pr_wait(uint64_t *bar, unsigned parity, RowsShared *sh, const KvView &kv) {
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

// Two f32 values as the packed 16-bit parts of an operand.  A part that is
// not finite is the whole value.
template <int TYPE, int N>
__device__ __forceinline__ void split2(float a, float b, unsigned (&part)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        float ra, rb;
        if constexpr (TYPE == KV_F16) {
            const __half2 h = __floats2half2_rn(a, b);
            part[i] = *reinterpret_cast<const unsigned *>(&h);
            const float2 f = __half22float2(h);
            ra = f.x, rb = f.y;
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            part[i] = *reinterpret_cast<const unsigned *>(&h);
            ra = __uint_as_float(part[i] << 16), rb = __uint_as_float(part[i] & 0xffff0000u);
        }
        if (i + 1 < N) {
            a = fabsf(ra) < INFINITY ? __fsub_rn(a, ra) : 0.f;
            b = fabsf(rb) < INFINITY ? __fsub_rn(b, rb) : 0.f;
        }
    }
}
// The same of two softmax weights (finite, or NaN: then the row is redone).
template <int TYPE, int N>
__device__ __forceinline__ void split2_weights(float a, float b, unsigned (&part)[N]) {
    if constexpr (TYPE == KV_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        const __half2 r = __floats2half2_rn(__fsub_rn(a, f.x), __fsub_rn(b, f.y));
        part[0] = *reinterpret_cast<const unsigned *>(&h);
        part[1] = *reinterpret_cast<const unsigned *>(&r);
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

// One row's keys [lo, hi) of the CTA's list on the CUDA cores, a warp per row:
// 32 keys at a time, a key per lane for the scores, head_dim over the lanes
// for the values.  Rows that met a value that is not finite are redone so:
// on the tensor cores 0 x NaN of a key that a row does not see would reach it.
struct RowState {
    float m, l, acc[4];
};
template <int TYPE>
__device__ __noinline__ RowState attend_row(const KvView &kv, const BatchView &b, int seq, int head, const float *q,
                                            float sl2, SeenKeys keys, int lo, int hi, int from, int sink_end, int to) {
    using T = typename KvElem<TYPE>::T;
    const int lane = threadIdx.x & 31, hd = kv.hd;
    RowState r;
    r.m = PR_NO_MAX;
    r.l = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) r.acc[c] = 0.f;
    if (hi > to) hi = to;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        long long off = -1;
        if (i < hi && (i < sink_end || i >= from)) off = key_offset(kv, b, seq, (unsigned)keys.key(i), head);
        float x = -INFINITY;
        if (off >= 0) {
            const T *k = reinterpret_cast<const T *>(kv.k) + off;
            float dot = 0.f;
            for (int d = 0; d < hd; d++) dot = __fmaf_rn(q[d], KvElem<TYPE>::get(k + d), dot);
            x = __fmul_rn(dot, sl2);
        }
        float top = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, r.m);
        const float f = ex2(__fsub_rn(r.m, top)), w = ex2(__fsub_rn(x, top));
        r.m = top;
        float total = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total = __fadd_rn(total, __shfl_xor_sync(0xffffffffu, total, o));
        r.l = __fmaf_rn(r.l, f, total);
#pragma unroll
        for (int c = 0; c < 4; c++) r.acc[c] = __fmul_rn(r.acc[c], f);
        for (int j = 0; j < 32; j++) {
            const long long o = __shfl_sync(0xffffffffu, off, j);
            const float wj = __shfl_sync(0xffffffffu, w, j);
            if (o < 0) continue;
            const T *v = reinterpret_cast<const T *>(kv.v) + o;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (lane + 32 * c < hd) r.acc[c] = __fmaf_rn(wj, KvElem<TYPE>::get(v + lane + 32 * c), r.acc[c]);
        }
    }
    return r;
}

template <int TYPE, int HDP>
__global__ void __launch_bounds__(PR_THREADS, 1)
    paged_rows_kernel(KvView kv, BatchView b, PagedAttnView a, RowsPlan plan) {
    using Cfg = RowsCfg<TYPE, HDP>;
    constexpr int KT = Cfg::KT, NQ = Cfg::NQ, NC = Cfg::NC, T = Cfg::T, RT = Cfg::RT;
    extern __shared__ __align__(1024) unsigned char pr_smem[];
    unsigned char *s_q = pr_smem;                   // [tile][part] operands of 128 rows
    unsigned char *s_kv = pr_smem + Cfg::QBYTES;    // ring of key / value tiles
    RowsShared *sh = reinterpret_cast<RowsShared *>(pr_smem + Cfg::SMEM - 3072);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.num_heads / kv.kv_heads, hd = kv.hd;
    if (smem_addr(pr_smem) & 1023u) {  // the swizzled tiles need it
        if (tid == 0) paged_flag(kv, PAGED_WAIT_GAVE_UP);
        return;
    }
    pdl_release();

    // rows that no sequence owns
    {
        const int end = b.row_start[b.num_seqs];
        for (long long r = (long long)(end < 0 ? 0 : end) + blockIdx.x; r < b.num_rows; r += gridDim.x)
            for (int e = tid; e < a.num_heads * hd; e += PR_THREADS) a.out[(size_t)r * a.ldo + e] = 0.f;
    }
    // this CTA's row tile: tiles are counted from the last sequence's last
    // (the longest under the causal mask) to the first
    const int split = blockIdx.x % plan.splits;
    const int head = blockIdx.x / plan.splits % kv.kv_heads;
    const int index = blockIdx.x / plan.splits / kv.kv_heads;
    if (warp == 0) {
        int before = 0, found = 0;
        for (int s0 = b.num_seqs - 1; s0 >= 0 && !found; s0 -= 32) {
            const int s = s0 - lane;
            int start = 0, rows = 0;
            if (s >= 0) {
                start = b.row_start[s];
                rows = b.row_start[s + 1] - start;
                if (start < 0 || rows < 0 || rows > b.num_rows - start) rows = 0;
            }
            const int n = (int)(((long long)rows * group + RT - 1) / RT);
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += t;
            }
            const bool here = index >= before + sum - n && index < before + sum;
            const unsigned who = __ballot_sync(0xffffffffu, here);
            if (here) {
                sh->seq = s;
                sh->row0 = start;
                sh->rows = rows;
                sh->tile = n - 1 - (index - (before + sum - n));
            }
            found = who != 0;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) sh->found = found;
    }
    __syncthreads();
    if (!sh->found) return;
    if (warp == 0) tc_alloc(&sh->taddr, PR_TMEM_COLS);
    if (tid == 32) {
        for (int i = 0; i < Cfg::NSLOT; i++) {
            mbar_init(&sh->full[i], PR_PRODUCERS);
            mbar_init(&sh->empty[i], 1);
        }
        for (int x = 0; x < 2; x++) {
            mbar_init(&sh->s_full[x], 1);
            mbar_init(&sh->p_full[x], 128);
            mbar_init(&sh->o_full[x], 1);
        }
        mbar_init(&sh->q_full, 256);
        mbar_init(&sh->drain, 1);
        sh->abort = 0;
        mbar_fence_init();
    }
    const int seq = sh->seq, row0 = sh->row0, rows = sh->rows, tile = sh->tile;
    const int pos0 = b.kv_len[seq] - rows;  // position of the sequence's first row
    // tokens of this tile, and the list of keys any of them sees
    const int tok0 = (int)((long long)tile * RT / group);
    const long long last_flat = (long long)tile * RT + RT - 1;
    const int tok1 = last_flat / group < rows ? (int)(last_flat / group) : rows - 1;
    const SeenKeys keys = seen_keys(pos0 + tok0, pos0 + tok1, a.window, a.sinks);
    const int all_tiles = (keys.n + KT - 1) / KT;
    const int per_split = (all_tiles + plan.splits - 1) / plan.splits;
    const int lo = split * per_split * KT;
    int hi = lo + per_split * KT;
    hi = hi < keys.n ? hi : keys.n;
    const int ntile = lo < hi ? (hi - lo + KT - 1) / KT : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned taddr = sh->taddr;

    if (warp < 8) {
        // ------------------------------------------------ q, softmax, output
        const int x = warp >> 2, r = tid & 127;      // stream, row of its tile
        const long long flat = (long long)tile * RT + (T == 2 ? x * 128 : 0) + r;
        const int tok = (int)(flat / group), h = head * group + (int)(flat % group);
        const bool row_ok = tok < rows;
        const int row = row0 + (row_ok ? tok : 0);
        const int pos = row_ok ? pos0 + tok : -1;
        // list positions this row sees: [0, sink_end) and [from, to)
        const int to = pos >= 0 ? pos - keys.low + keys.sinks + 1 : 0;
        const int sink_end = a.sinks < 0x7fffffffu ? (int)a.sinks : 0x7fffffff;
        int from = 0;
        if (a.window != 0 && pos >= 0 && (unsigned)pos >= a.window) from = pos - (int)a.window + 1 - keys.low + keys.sinks;
        float sl2 = __fmul_rn(a.scale, 1.44269504088896340736f);
        {
            const float *src = a.q + (size_t)row * a.ldq + (size_t)h * hd;
            const bool vec = (((uintptr_t)a.q | (a.ldq * 4)) & 15) == 0;
            float up = 1.0f;
            if constexpr (Cfg::F16) {
                float top = 0.f;
                if (row_ok)
                    for (int d = 0; d < hd; d++) top = fmaxf(top, fabsf(src[d]));
                if (top > 0.f && top < INFINITY) {
                    int e;
                    frexpf(top, &e);  // top = f 2^e, 0.5 <= f < 1
                    e = 15 - e;
                    e = e > 120 ? 120 : e < -120 ? -120 : e;
                    up = __uint_as_float((unsigned)(127 + e) << 23);
                    sl2 = __fmul_rn(sl2, __uint_as_float((unsigned)(127 - e) << 23));
                }
            }
            unsigned char *tq = s_q + (T == 2 ? x * NQ * Cfg::QPART : 0);
            // with one tile the two warpgroups take alternate chunks of it
            for (int c = T == 2 ? 0 : x; c < HDP / 8; c += T == 2 ? 1 : 2) {
                float f[8];
                const bool in = row_ok && c * 8 < hd;
                if (in && vec) {
                    const float4 u = *reinterpret_cast<const float4 *>(src + c * 8);
                    const float4 w = *reinterpret_cast<const float4 *>(src + c * 8 + 4);
                    f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = w.x, f[5] = w.y, f[6] = w.z, f[7] = w.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) f[i] = in ? src[c * 8 + i] : 0.f;
                }
                unsigned part[4][NQ];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    split2<TYPE, NQ>(__fmul_rn(f[2 * i], up), __fmul_rn(f[2 * i + 1], up), part[i]);
                const unsigned o = sw16_off(r, c, 128);
#pragma unroll
                for (int p = 0; p < NQ; p++)
                    *reinterpret_cast<uint4 *>(tq + p * Cfg::QPART + o) =
                        make_uint4(part[0][p], part[1][p], part[2][p], part[3][p]);
            }
            fence_async_smem();
            mbar_arrive(&sh->q_full);
        }
        const unsigned t_s = taddr + ((unsigned)((warp & 3) * 32) << 16) + (unsigned)(x * Cfg::STREAM);
        const unsigned t_o = t_s + Cfg::SP;
        float m = PR_NO_MAX, l = 0.f;
        bool ok = true, any = false;
        unsigned phase = 0;
        for (int j = T == 2 ? 0 : x; j < ntile; j += T == 2 ? 1 : 2) {
            ok = __all_sync(0xffffffffu, pr_wait(&sh->s_full[x], phase, sh, kv));  // TMEM loads are warp-wide
            if (!ok) break;
            phase ^= 1;
            tc_fence_after();
            float v[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 32) tmem_ld32(t_s + c, v + c);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < KT; c += 32) pin32(v + c);
            const int i0 = lo + j * KT;
            bool whole = i0 + KT <= to && i0 + KT <= hi && (i0 + KT <= sink_end || i0 >= from);
#pragma unroll
            for (int c = 0; c < KT / 32; c++) whole = whole && sh->valid[j & 7][c] == 0xffffffffu;
            if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
                for (int c = 0; c < KT; c++) {
                    const int i = i0 + c;
                    const bool seen = i < to && (i < sink_end || i >= from) && ((sh->valid[j & 7][c >> 5] >> (c & 31)) & 1u);
                    v[c] = seen ? v[c] : -INFINITY;
                }
            }
            float t0 = v[0], t1 = v[1], t2 = v[2], t3 = v[3];
#pragma unroll
            for (int c = 4; c < KT; c += 4) {
                t0 = fmaxf(t0, v[c]);
                t1 = fmaxf(t1, v[c + 1]);
                t2 = fmaxf(t2, v[c + 2]);
                t3 = fmaxf(t3, v[c + 3]);
            }
            const float top = __fmul_rn(fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)), sl2);
            const bool move = top > m + PR_RESCALE;
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? ex2(__fsub_rn(m, top)) : 1.0f;
                m = move ? top : m;
                l = __fmul_rn(l, f);
                if (any) {  // the stream's earlier products are complete: so are its scores
#pragma unroll 1
                    for (int c = 0; c < HDP; c += 8) tmem_scale8(t_o + c, f);  // few registers: the scores are live
                }
            }
            any = true;
            float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
            // the scores are all in registers: the weights' parts take their place
#pragma unroll
            for (int c = 0; c < KT; c += 32) {
                unsigned w[NQ][16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float e0 = ex2(__fmaf_rn(v[c + i], sl2, -m)), e1 = ex2(__fmaf_rn(v[c + i + 1], sl2, -m));
                    const float e2 = ex2(__fmaf_rn(v[c + i + 2], sl2, -m)), e3 = ex2(__fmaf_rn(v[c + i + 3], sl2, -m));
                    l0 = __fadd_rn(l0, e0);
                    l1 = __fadd_rn(l1, e1);
                    l2 = __fadd_rn(l2, e2);
                    l3 = __fadd_rn(l3, e3);
                    unsigned p[NQ], q[NQ];
                    split2_weights<TYPE, NQ>(e0, e1, p);
                    split2_weights<TYPE, NQ>(e2, e3, q);
#pragma unroll
                    for (int n = 0; n < NQ; n++) w[n][i / 2] = p[n], w[n][i / 2 + 1] = q[n];
                }
#pragma unroll
                for (int n = 0; n < NQ; n++) tmem_st16(t_s + n * (KT / 2) + c / 2, w[n]);
            }
            l = __fadd_rn(l, __fadd_rn(__fadd_rn(l0, l1), __fadd_rn(l2, l3)));
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&sh->p_full[x]);
        }
        if (ok && any) ok = __all_sync(0xffffffffu, pr_wait(&sh->o_full[x], 0, sh, kv));
        tc_fence_after();
        float *s_o = reinterpret_cast<float *>(s_q);  // [head_dim][128]: the odd stream's sums
        if constexpr (T == 1) {
            // the q tiles are free: every q.k product is complete once o_full[1]
            // is, and with fewer than two key tiles there is no odd stream
            if (x == 1) {
                if (ok && any) {
#pragma unroll 1
                    for (int c = 0; c < HDP; c += 32) {
                        float o[32];
                        tmem_ld32(t_o + c, o);
                        tmem_wait_ld();
                        pin32(o);
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c + i < hd) s_o[(c + i) * 128 + r] = o[i];
                    }
                }
                sh->ml[0][r] = m;
                sh->ml[1][r] = l;
            }
            if (named_bar_or(2, 256, !ok)) ok = false;
        }
        if (ok && (T == 2 || x == 0)) {
            float mine = 1.0f, other = 0.f;
            if constexpr (T == 1) {
                const float m1 = sh->ml[0][r], l1 = sh->ml[1][r];
                const float top = fmaxf(m, m1);
                mine = ex2(__fsub_rn(m, top));
                other = ex2(__fsub_rn(m1, top));
                l = __fadd_rn(__fmul_rn(l, mine), __fmul_rn(l1, other));
                m = top;
            }
            const bool two = T == 1 && ntile > 1;
            const bool whole = plan.splits == 1;
            const float inv = !whole ? 1.0f : l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
            const size_t part = ((size_t)row * a.num_heads + h) * plan.splits + split;
            float *dst = whole ? a.out + (size_t)row * a.ldo + (size_t)h * hd : plan.part_o + part * hd;
            const bool vec = !whole || (((uintptr_t)a.out | (a.ldo * 4)) & 15) == 0;
            bool finite = fabsf(l) < INFINITY;
#pragma unroll 1
            for (int c = 0; c < HDP; c += 32) {
                float o[32];
                if (any) {
                    tmem_ld32(t_o + c, o);
                    tmem_wait_ld();
                    pin32(o);
                }
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    float y = any ? o[i] : 0.f;
                    if constexpr (T == 1) {
                        y = __fmul_rn(y, mine);
                        if (two && c + i < hd) y = __fmaf_rn(s_o[(c + i) * 128 + r], other, y);
                    }
                    y = __fmul_rn(y, inv);
                    if (c + i < hd) finite = finite && fabsf(y) < INFINITY;
                    o[i] = y;
                }
                if (row_ok) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        if (c + i >= hd) continue;
                        if (vec)
                            *reinterpret_cast<float4 *>(dst + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        else
#pragma unroll
                            for (int u = 0; u < 4; u++) dst[c + i + u] = o[i + u];
                    }
                }
            }
            if (!whole && row_ok) plan.part_ml[part] = make_float2(m, l);
            unsigned redo = __ballot_sync(0xffffffffu, row_ok && !finite);
            __syncwarp();
            while (redo) {
                const int who = __ffs(redo) - 1;
                redo &= redo - 1;
                const int rrow = __shfl_sync(0xffffffffu, row, who), rh = __shfl_sync(0xffffffffu, h, who);
                const int rfrom = __shfl_sync(0xffffffffu, from, who), rto = __shfl_sync(0xffffffffu, to, who);
                const RowState st = attend_row<TYPE>(kv, b, seq, head, a.q + (size_t)rrow * a.ldq + (size_t)rh * hd,
                                                     __fmul_rn(a.scale, 1.44269504088896340736f), keys, lo, hi, rfrom,
                                                     sink_end, rto);
                const size_t at = ((size_t)rrow * a.num_heads + rh) * plan.splits + split;
                float *d = whole ? a.out + (size_t)rrow * a.ldo + (size_t)rh * hd : plan.part_o + at * hd;
                const float div = whole ? st.l : 1.0f;
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (lane + 32 * c < hd) d[lane + 32 * c] = div == 0.f ? 0.f : __fdiv_rn(st.acc[c], div);
                if (!whole && lane == 0) plan.part_ml[at] = make_float2(st.m, st.l);
            }
        }
    } else if (warp == 8) {
        // --------------------------------------------------------- the MMAs
        if (lane == 0 && ntile > 0) {
            const unsigned idesc_s = umma_idesc_f16(TYPE != KV_F16, 128, KT, false);
            const unsigned idesc_o = umma_idesc_f16(TYPE != KV_F16, 128, (hd + 15) / 16 * 16, true);
            const int qk_steps = (hd + 15) / 16;
            const unsigned a_q = smem_addr(s_q), a_kv = smem_addr(s_kv);
            unsigned n_take = 0;  // slots taken so far
            bool ok = pr_wait(&sh->q_full, 0, sh, kv);
            auto take = [&]() -> int {  // the next slot, filled
                const int slot = (int)(n_take % Cfg::NSLOT);
                ok = ok && pr_wait(&sh->full[slot], (n_take / Cfg::NSLOT) & 1u, sh, kv);
                n_take++;
                return slot;
            };
            // the products of parts that count, the smallest first: each MMA
            // cuts its sum at the last bit of the largest addend
            auto parts = [&](auto f) {
                if constexpr (NC == 1) {
#pragma unroll
                    for (int i = NQ - 1; i >= 0; i--) f(i, 0, i == NQ - 1);
                } else {
                    f(2, 0, true), f(0, 2, false), f(1, 1, false), f(1, 0, false), f(0, 1, false), f(0, 0, false);
                }
            };
            auto scores = [&](int x, int slot) {
                const uint64_t dq = umma_desc_sw128(a_q + (T == 2 ? x * NQ * Cfg::QPART : 0));
                const uint64_t dk = umma_desc_sw128(a_kv + slot * Cfg::SLOT);
                parts([&](int i, int c, bool first) {
                    for (int ks = 0; ks < qk_steps; ks++) {
                        const unsigned ao = i * Cfg::QPART + (ks >> 2) * 128 * 128 + (ks & 3) * 32;
                        const unsigned bo = c * Cfg::PART + (ks >> 2) * KT * 128 + (ks & 3) * 32;
                        tc_mma_f16(taddr + x * Cfg::STREAM, dq + (ao >> 4), dk + (bo >> 4), idesc_s, !first || ks > 0);
                    }
                });
            };
            auto values = [&](int x, int slot, bool acc) {
                const uint64_t dv = umma_desc_sw128_mn(a_kv + slot * Cfg::SLOT, KT * 128);
                parts([&](int i, int c, bool first) {
#pragma unroll
                    for (int ks = 0; ks < KT / 16; ks++)
                        tc_mma_f16_ta(taddr + x * Cfg::STREAM + Cfg::SP, taddr + x * Cfg::STREAM + i * (KT / 2) + ks * 8,
                                      dv + ((c * Cfg::PART + ks * 2048) >> 4), idesc_o, acc || !first || ks > 0);
                });
            };
            if constexpr (T == 2) {
                int k = take();
                if (ok) {
                    tc_fence_after();
                    scores(0, k);
                    tc_commit(&sh->s_full[0]);
                    scores(1, k);
                    tc_commit(&sh->s_full[1]);
                    tc_commit(&sh->empty[k]);
                }
                for (int j = 0; j < ntile && ok; j++) {
                    const int v = take();
                    k = -1;
                    for (int x = 0; x < 2 && ok; x++) {
                        ok = ok && pr_wait(&sh->p_full[x], j & 1u, sh, kv);
                        if (!ok) break;
                        tc_fence_after();
                        values(x, v, j > 0);
                        if (j + 1 < ntile) {
                            if (x == 0) k = take();
                            if (!ok) break;
                            tc_fence_after();
                            scores(x, k);
                            tc_commit(&sh->s_full[x]);
                        } else {
                            tc_commit(&sh->o_full[x]);
                        }
                    }
                    if (!ok) break;
                    tc_commit(&sh->empty[v]);
                    if (k >= 0) tc_commit(&sh->empty[k]);
                }
            } else {
                for (int j = 0; j < 2 && j < ntile && ok; j++) {
                    const int k = take();
                    if (!ok) break;
                    tc_fence_after();
                    scores(j, k);
                    tc_commit(&sh->s_full[j]);
                    tc_commit(&sh->empty[k]);
                }
                for (int j = 0; j < ntile && ok; j++) {
                    const int x = j & 1, v = take();
                    ok = ok && pr_wait(&sh->p_full[x], (j >> 1) & 1u, sh, kv);
                    if (!ok) break;
                    tc_fence_after();
                    values(x, v, j > 1);
                    tc_commit(&sh->empty[v]);
                    if (j + 2 < ntile) {
                        const int k = take();
                        if (!ok) break;
                        tc_fence_after();
                        scores(x, k);
                        tc_commit(&sh->s_full[x]);
                        tc_commit(&sh->empty[k]);
                    } else {
                        tc_commit(&sh->o_full[x]);
                    }
                }
            }
            // what was issued has to end before the TMEM is freed
            tc_commit(&sh->drain);
            const long long t0 = clock64();
            while (!mbar_test(&sh->drain, 0) && clock64() - t0 < WAIT_LIMIT) {
            }
        }
    } else {
        // ------------------------------------------- keys and values to slots
        const int p = tid - 9 * 32;
        constexpr int NOFF = 128 / KT;  // tiles whose offsets are kept
        constexpr int CH = HDP / 8;     // 16-byte chunks of a row's part
        const int in_chunks = (hd + 15) / 16 * 2;  // chunks a product reads
        unsigned n_put = 0;
        int pending = -1;  // slot whose copies are under way
        bool ok = true;
        auto land = [&]() {
            if (pending < 0) return;
            cp_async_wait<0>();
            fence_async_smem();
            mbar_arrive(&sh->full[pending]);
            pending = -1;
        };
        // offsets of tile j's keys; the barriers order them with the copies
        auto lookup = [&](int j) {
            for (int i = p; i < KT; i += PR_PRODUCERS) {
                const int at = lo + j * KT + i;
                sh->off[(j % NOFF) * KT + i] = at < hi ? key_offset(kv, b, seq, (unsigned)keys.key(at), head) : -1;
            }
            named_bar_sync(1, PR_PRODUCERS);
            if (p < KT / 32) {
                unsigned bits = 0;
                for (int i = 0; i < 32; i++) bits |= (sh->off[(j % NOFF) * KT + p * 32 + i] >= 0 ? 1u : 0u) << i;
                sh->valid[j & 7][p] = bits;
            }
        };
        auto put = [&](int j, const void *pool) {
            const int slot = (int)(n_put % Cfg::NSLOT);
            if (n_put >= (unsigned)Cfg::NSLOT) {
                const unsigned par = (n_put / Cfg::NSLOT - 1) & 1u;
                if (!mbar_test(&sh->empty[slot], par)) {
                    land();
                    ok = pr_wait(&sh->empty[slot], par, sh, kv);
                }
            }
            n_put++;
            if (!ok) return;
            const long long *off = sh->off + (j % NOFF) * KT;
            unsigned char *dst = s_kv + slot * Cfg::SLOT;
            if constexpr (TYPE != KV_F32) {
                for (int e = p; e < KT * CH; e += PR_PRODUCERS) {
                    const int r = e / CH, c = e % CH;
                    if (c >= in_chunks) continue;
                    const long long o = off[r];
                    const bool in = o >= 0 && c * 8 < hd;
                    const char *src = reinterpret_cast<const char *>(pool) + (in ? (size_t)o * 2 + c * 16 : 0);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(dst) + sw16_off(r, c, KT)),
                                 "l"(src), "r"(in ? 16u : 0u));
                }
                cp_async_commit();
                if (pending >= 0) {
                    cp_async_wait<1>();
                    fence_async_smem();
                    mbar_arrive(&sh->full[pending]);
                }
                pending = slot;
            } else {
                constexpr int PER = (KT * CH + PR_PRODUCERS - 1) / PR_PRODUCERS;
                float4 u[PER][2];
#pragma unroll
                for (int n = 0; n < PER; n++) {
                    const int e = p + n * PR_PRODUCERS, r = e / CH, c = e % CH;
                    const long long o = e < KT * CH ? off[r] : -1;
                    if (o >= 0 && c * 8 < hd) {
                        const float4 *src = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(pool) + o + c * 8);
                        u[n][0] = src[0];
                        u[n][1] = src[1];
                    } else {
                        u[n][0] = u[n][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
#pragma unroll
                for (int n = 0; n < PER; n++) {
                    const int e = p + n * PR_PRODUCERS, r = e / CH, c = e % CH;
                    if (e >= KT * CH || c >= in_chunks) continue;
                    unsigned part[4][3];
                    split2<KV_BF16, 3>(u[n][0].x, u[n][0].y, part[0]);
                    split2<KV_BF16, 3>(u[n][0].z, u[n][0].w, part[1]);
                    split2<KV_BF16, 3>(u[n][1].x, u[n][1].y, part[2]);
                    split2<KV_BF16, 3>(u[n][1].z, u[n][1].w, part[3]);
                    const unsigned at = sw16_off(r, c, KT);
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        *reinterpret_cast<uint4 *>(dst + i * Cfg::PART + at) =
                            make_uint4(part[0][i], part[1][i], part[2][i], part[3][i]);
                }
                fence_async_smem();
                mbar_arrive(&sh->full[slot]);
            }
        };
        if constexpr (T == 2) {
            for (int j = 0; j < ntile && ok; j++) {
                lookup(j);
                named_bar_sync(1, PR_PRODUCERS);
                put(j, kv.k);
                if (ok) put(j, kv.v);
                ok = !named_bar_or(1, PR_PRODUCERS, !ok);
            }
        } else {
            for (int j = 0; j <= ntile && ok && ntile > 0; j++) {
                if (j < ntile) {
                    lookup(j);
                    named_bar_sync(1, PR_PRODUCERS);
                    put(j, kv.k);
                }
                if (j > 0 && ok) put(j - 1, kv.v);
                ok = !named_bar_or(1, PR_PRODUCERS, !ok);
            }
        }
        land();
        cp_async_wait<0>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tc_dealloc(taddr, PR_TMEM_COLS);
}

template <int TYPE, int HDP>
void go(const KvView &kv, const BatchView &b, const PagedAttnView &a, const RowsPlan &plan, cudaStream_t s) {
    static SmemOptIn opt;
    opt(paged_rows_kernel<TYPE, HDP>, RowsCfg<TYPE, HDP>::SMEM);
    const unsigned grid = (unsigned)(plan.tiles * kv.kv_heads * plan.splits);
    launch_kernel(paged_rows_kernel<TYPE, HDP>, dim3(grid), dim3(PR_THREADS), RowsCfg<TYPE, HDP>::SMEM, s, false, kv, b, a,
                  plan);
}

}  // namespace

RowsPlan plan_paged_rows(const KvView &kv, const BatchView &b, const PagedAttnView &a, uint32_t max_kv_len) {
    RowsPlan p{};
    const uint64_t group = a.num_heads / kv.kv_heads;
    const uint64_t rt = kv.type == KV_F16 ? 256 : 128, kt = kv.type == KV_F16 ? 128 : 64;
    // a tile may end inside each sequence: an upper bound of their number
    p.tiles = (uint64_t)b.num_rows * group / rt + (uint64_t)std::min(b.num_seqs, b.num_rows);
    const uint64_t units = std::max<uint64_t>(p.tiles * kv.kv_heads, 1);
    uint64_t most = max_kv_len;
    if (a.window) most = std::min<uint64_t>(most, (uint64_t)a.window + a.sinks + rt / group + 1);
    const uint64_t key_tiles = (most + kt - 1) / kt;
    // fewer tiles than SMs: split the keys, at least four key tiles each
    uint64_t splits = units < 148 ? std::min<uint64_t>(148 / units, key_tiles / 4) : 1;
    p.splits = (int)std::max<uint64_t>(splits, 1);
    const uint64_t parts = (uint64_t)b.num_rows * a.num_heads * p.splits;
    p.ml_bytes = p.splits > 1 ? (parts * sizeof(float2) + 15) / 16 * 16 : 0;
    p.scratch_bytes = p.splits > 1 ? p.ml_bytes + parts * kv.hd * sizeof(float) : 0;
    return p;
}

void launch_paged_rows(const KvView &kv, const BatchView &b, const PagedAttnView &a, const RowsPlan &plan, cudaStream_t s) {
    if (kv.type == KV_F32)
        kv.hd <= 64 ? go<KV_F32, 64>(kv, b, a, plan, s) : go<KV_F32, 128>(kv, b, a, plan, s);
    else if (kv.type == KV_F16)
        kv.hd <= 64 ? go<KV_F16, 64>(kv, b, a, plan, s) : go<KV_F16, 128>(kv, b, a, plan, s);
    else
        kv.hd <= 64 ? go<KV_BF16, 64>(kv, b, a, plan, s) : go<KV_BF16, 128>(kv, b, a, plan, s);
    if (plan.splits > 1) launch_paged_join(kv, b, a, plan.part_ml, plan.part_o, 0, plan.splits, s);
}

}  // namespace slm
