// kernels_paged_rows.cu -- attention of several new rows per sequence (a
// prompt, or a chunk behind an earlier context) over the paged cache, on the
// tcgen05 tensor cores at f32 accuracy.
//
// The tensor cores multiply 16-bit operands exactly and add in f32, so an f32
// operand is written as a sum of 16-bit parts and the products of the parts
// are added up:
//   f16 pages:  q 2^e = q0 + q1 / 2^12 (e per row, so that the row's largest
//               element is near 2^15), w = w0 + w1 / 2^12 for the softmax weights
//               w <= 2^15; 2 products each for q.k and w.v, the second parts'
//               first and the others onto them as the MMA takes D / 2^12.
//   bf16 pages: three bf16 parts of q and w (24 bits), 3 products each.
//   f32 pages:  three bf16 parts of q, w, k and v; the 6 products whose size
//               is above 2^-24 of the leading one.
//
// The tensor core cuts each sum at the last bit of its largest addend, always
// towards zero: about 2e-8 of the sum per MMA, which over the hundreds of MMAs
// of a long row adds up.  So no chain of MMAs is longer than one key tile (8 to
// 24, 48 for q.k of f32 pages with head_dim above 64; the smallest products
// first): every tile's w.v goes to TMEM afresh and is added to the row's sums in
// registers.  Against 64 bits, in the 2-norm, 300 rows behind 3000 keys are off by
// 2e-7 to 7e-7 with q of N(0, 1) and 1.5 times it, and by 5e-7 (head_dim 64) and 8e-7
// (f32 and bf16 pages, 128) or 1.1e-6 (f16, 128) with q sixteen times as large,
// where f32 arithmetic itself gives 1.7e-6 and 2.6e-6.
//
// A CTA takes 128 rows of one (sequence, KV head), the query heads of the KV
// head side by side (row = token * group + head in group), so every key read
// serves all of them.  Warps 0-7 run the softmax: thread r and r + 128 hold
// the two halves of row r's keys of a tile, and of its head_dim.  Warp 8
// issues the MMAs, warps 9-11 (9-15 for f32 pages) bring keys and values from
// the pages into a ring of shared-memory slots.  Scores and tile results are double-buffered in
// TMEM: q.k of tile j + 1 and w.v of tile j - 1 run under the softmax of j.
#include "async.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace slm {

namespace {

constexpr unsigned PR_TMEM_COLS = 512;

template <int TYPE, int HDP>
struct RowsCfg {
    static constexpr bool F16 = TYPE == KV_F16;
    static constexpr int KT = F16 ? 128 : 64;    // keys per tile
    static constexpr int NQ = F16 ? 2 : 3;       // parts of q and of the weights
    static constexpr int NC = TYPE == KV_F32 ? 3 : 1;  // parts of k and v
    // warps 0-7 and 8, and those that copy: f32 pages are split into parts on
    // the way, and three warps of it held the rest up (16 chunks of up to 512 rows
    // behind up to 2048 keys: 178 us, with seven 146)
    static constexpr int PRODUCERS = TYPE == KV_F32 ? 224 : 96, THREADS = 288 + PRODUCERS;
    static constexpr int R_LAUNCH = TYPE == KV_F32 ? 128 : 168;  // registers of a thread at launch, and after the split
    static constexpr int R_SOFTMAX = F16 ? 200 : TYPE == KV_F32 ? 152 : 184, R_OTHER = F16 ? 104 : TYPE == KV_F32 ? 104 : 136;
    static_assert(256 * R_SOFTMAX + (THREADS - 256) * R_OTHER == THREADS * R_LAUNCH, "registers");
    static constexpr int PART = KT * HDP * 2;    // bytes of one part of a key tile
    static constexpr int SLOT = PART * NC;
    static constexpr int QPART = 128 * HDP * 2;
    static constexpr int QBYTES = NQ * QPART;
    // k and v of even and of odd tiles (one tile where f32 pages leave no room
    // for two): the MMAs' operands are the same every second tile
    static constexpr int NSLOT = TYPE == KV_F32 && HDP == 128 ? 2 : 4;
    // TMEM columns: score / weight buffers (128 or 3 x 32 used) at 0 and 128,
    // results at 256 and 256 + HDP
    static constexpr int T_S = 128, T_O = 256;
    static constexpr int BIG = QBYTES + NSLOT * SLOT;
    // at least 120 KB: one CTA per SM, whose TMEM it takes whole
    static constexpr int SMEM = (BIG > 120 * 1024 ? BIG : 120 * 1024) + 3072;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(T_O + 2 * HDP <= (int)PR_TMEM_COLS && KT <= T_S && NQ * KT / 2 <= T_S, "TMEM");
};

// The small shared data, after the tiles.
struct RowsShared {
    uint64_t full[4], empty[4], s_full[2], p_full[2], o_full[2], q_full, seen_all, swapped, drain;
    long long off[128];       // byte offsets of the newest tile's keys
    unsigned valid[8][4];     // held keys of the newest 8 tiles
    float row[2][128];        // exchanged between the halves of a row; 2^-e of q's rows before
    int move[4];              // some row's reference has to move, by tile
    unsigned taddr;
    int abort;
    // the CTA's work
    int seq, row0, rows, past, tile, found, bits;  // row0: first activation row of the sequence
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
__host__ __device__ constexpr unsigned umma_idesc_f16(bool bf16, int M, int N, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24);
}
// D[128 x N] (+)= A[128 x 16] B[N x 16]^T, A in shared memory or in TMEM, called
// by the whole warp.  (With the election inside, 128-wide MMAs issue every 64
// cycles, their full rate, and 64-wide ones every 49; with a predicate kept
// in a register every 73.)
__device__ __forceinline__ void tc_mma_f16(unsigned d, uint64_t adesc, uint64_t bdesc, unsigned idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"((unsigned)acc)
        : "memory");
}
// The same on top of D / 2^12: D holds the products of the second f16 parts.
static_assert(F16_PART2_LOG2 == 12, "the immediate below");
__device__ __forceinline__ void tc_mma_f16_onto_part2(unsigned d, uint64_t adesc, uint64_t bdesc, unsigned idesc) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.eq.u32 p, 0, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 12;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc)
        : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ta_onto_part2(unsigned d, unsigned a, uint64_t bdesc, unsigned idesc) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.eq.u32 p, 0, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, 12;\n}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc)
        : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ta(unsigned d, unsigned a, uint64_t bdesc, unsigned idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"((unsigned)acc)
        : "memory");
}
// What the copies wrote, before the lane that issues has the tensor core read
// it (by all 32 lanes after every wait it stood for about 1000 cycles a tile).
__device__ __forceinline__ void fence_async_elected() {
    asm volatile(
        "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n @q fence.proxy.async.shared::cta;\n}\n" ::: "memory");
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

// One arrival for a warp's 32 threads (an arrival of each is worked off one by
// one: at 256 a tile they took longer than the arithmetic).
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

template <int TYPE, int HDP>
__global__ void __launch_bounds__(RowsCfg<TYPE, HDP>::THREADS, 1)
    paged_rows_kernel(KvView kv, BatchView b, PagedAttnView a, RowsPlan plan) {
    using Cfg = RowsCfg<TYPE, HDP>;
    using Range = WeightRange<TYPE>;
    constexpr int KT = Cfg::KT, NQ = Cfg::NQ, NC = Cfg::NC;
    constexpr int CT = KT / 2, OC = HDP / 2;        // a thread's keys of a tile, and its part of head_dim
    extern __shared__ __align__(1024) unsigned char pr_smem[];
    unsigned char *s_q = pr_smem;                   // [part] operands of 128 rows
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
        const int start = min(max(b.row_start[0], 0), b.num_rows);
        const int end = min(max(b.row_start[b.num_seqs], start), b.num_rows);
        for (long long i = blockIdx.x; i < (long long)b.num_rows - end + start; i += gridDim.x) {
            const long long r = i < start ? i : i - start + end;
            for (int e = tid; e < a.num_heads * hd; e += Cfg::THREADS) a.out[(size_t)r * a.ldo + e] = 0.f;
        }
    }
    // this CTA's row tile: tiles are counted from the last sequence's last
    // (the longest under the causal mask) to the first
    const int split = blockIdx.x % plan.splits;
    const int head = blockIdx.x / plan.splits % kv.kv_heads;
    const int index = blockIdx.x / plan.splits / kv.kv_heads;
    if (warp == 0) {
        int before = 0, found = 0;
        bool bad = b.row_start[0] < 0 || b.row_start[b.num_seqs] > b.num_rows;
        // (the first CTA goes over all sequences, for the check)
        for (int s0 = b.num_seqs - 1; s0 >= 0 && (!found || blockIdx.x == 0); s0 -= 32) {
            const int s = s0 - lane;
            int start = 0, rows = 0, past = 0;  // rows of the sequence in the call, and past its end
            if (s >= 0) {
                start = b.row_start[s];
                const int end = b.row_start[s + 1];
                bad = bad || end < start;
                if (start >= 0 && start <= end) {
                    rows = max(min(end, b.num_rows) - start, 0);
                    past = end - start - rows;
                }
            }
            const int n = (int)(((long long)rows * group + 127) >> 7);
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
                sh->past = past;
                sh->tile = n - 1 - (index - (before + sum - n));
            }
            found |= who != 0;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) sh->found = found, sh->bits = bad ? PAGED_BAD_ROWS : 0;
    }
    __syncthreads();
    if (!sh->found) {
        if (tid == 0 && sh->bits) paged_flag(kv, sh->bits);
        return;
    }
    if (warp == 0) tc_alloc(&sh->taddr, PR_TMEM_COLS);
    if (tid == 32) {
        for (int i = 0; i < Cfg::NSLOT; i++) {
            mbar_init(&sh->full[i], Cfg::PRODUCERS);
            mbar_init(&sh->empty[i], 1);
        }
        for (int x = 0; x < 2; x++) {
            mbar_init(&sh->s_full[x], 1);
            mbar_init(&sh->p_full[x], 8);
            mbar_init(&sh->o_full[x], 1);
        }
        mbar_init(&sh->q_full, 8);
        mbar_init(&sh->seen_all, 8);
        mbar_init(&sh->swapped, 8);
        for (int i = 0; i < 4; i++) sh->move[i] = 0;
        mbar_init(&sh->drain, 1);
        sh->abort = 0;
        mbar_fence_init();
    }
    const int seq = sh->seq, row0 = sh->row0, rows = sh->rows, tile = sh->tile;
    const int pos0 = b.kv_len[seq] - rows - sh->past;  // position of the sequence's first row
    // tokens of this tile, and the list of keys any of them sees
    const unsigned flat0 = (unsigned)tile * 128u;
    const int tok0 = (int)(flat0 / (unsigned)group);
    int tok1 = (int)((flat0 + 127u) / (unsigned)group);
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
        if (warp == 0) tc_dealloc(sh->taddr, PR_TMEM_COLS);
        return;
    }
    constexpr unsigned taddr = 0;

    // the softmax threads keep a tile's scores and the row's sums in registers:
    // they take some of the others'
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(Cfg::R_SOFTMAX));
        // ------------------------------------------------ q, softmax, output
        const float sl2_all = __fmul_rn(a.scale, 1.44269504088896340736f);
        {  // a warp per row, its sixteen rows' loads in flight together
            const bool vec = (((uintptr_t)a.q | (a.ldq * 4)) & 15) == 0;
            const int c4 = lane * 4;
            // lane i < 16: the offset of the warp's row i in q, and whether it is one
            const unsigned my_flat = flat0 + (unsigned)(warp * 16 + (lane & 15)), my_tok = my_flat / (unsigned)group;
            const bool my_ok = (int)my_tok < rows;
            const long long my_at = my_ok ? (long long)((size_t)(row0 + (int)my_tok) * a.ldq +
                                                        (size_t)(head * group + (int)(my_flat - my_tok * (unsigned)group)) * hd)
                                          : (long long)((size_t)row0 * a.ldq);
            const unsigned oks = __ballot_sync(0xffffffffu, my_ok);
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += 16) {
                float f[16][4];
                const int c_in = c4 < hd ? c4 : 0;  // every load is of some row's element: none is held up by a branch
                if (vec) {
#pragma unroll
                    for (int u = 0; u < 16; u++) {
                        const float4 t = *reinterpret_cast<const float4 *>(a.q + __shfl_sync(0xffffffffu, my_at, r0 + u) + c_in);
                        f[u][0] = t.x, f[u][1] = t.y, f[u][2] = t.z, f[u][3] = t.w;
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 16; u++) {
                        const float *src = a.q + __shfl_sync(0xffffffffu, my_at, r0 + u) + c_in;
#pragma unroll
                        for (int i = 0; i < 4; i++) f[u][i] = src[i];
                    }
                }
#pragma unroll
                for (int u = 0; u < 16; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) f[u][i] = ((oks >> (r0 + u)) & 1u) && c4 < hd ? f[u][i] : 0.f;
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const int r = warp * 16 + r0 + u;
                    if constexpr (Cfg::F16) {
                        // the bits of non-negative floats order as they do
                        unsigned top = __float_as_uint(fabsf(f[u][0]));
#pragma unroll
                        for (int i = 1; i < 4; i++) top = max(top, __float_as_uint(fabsf(f[u][i])));
                        top = __reduce_max_sync(0xffffffffu, top);
                        int e = 141 - (int)(top >> 23);  // 2^14 <= top 2^e < 2^15
                        e = top == 0 || top >= 0x7f800000u ? 0 : e > 120 ? 120 : e;
                        const float up = __uint_as_float((unsigned)(127 + e) << 23);
                        if (lane == 0) sh->row[0][r] = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
                        for (int i = 0; i < 4; i++) f[u][i] = __fmul_rn(f[u][i], up);
                    }
                    if (c4 < HDP) {
                        unsigned p[NQ], q[NQ];
                        split2<TYPE, NQ>(f[u][0], f[u][1], p);
                        split2<TYPE, NQ>(f[u][2], f[u][3], q);
                        const unsigned o = sw16_off(r, lane >> 1, 128) + (lane & 1) * 8;
#pragma unroll
                        for (int i = 0; i < NQ; i++)
                            *reinterpret_cast<uint2 *>(s_q + i * Cfg::QPART + o) = make_uint2(p[i], q[i]);
                    }
                }
            }
            fence_async_smem();
            warp_arrive(&sh->q_full);
            if constexpr (Cfg::F16) named_bar_sync(2, 256);  // the rows' 2^-e
        }
        const int x = warp >> 2, r = tid & 127;  // half, row of the tile
        const unsigned flat = flat0 + (unsigned)r;
        const int tok = (int)(flat / (unsigned)group), h = head * group + (int)(flat % (unsigned)group);
        const bool row_ok = tok < rows;
        const int row = row0 + (row_ok ? tok : 0);
        const int pos = row_ok ? pos0 + tok : -1;
        // list positions this row sees: [0, sink_end) and [from, to)
        const int to = pos >= 0 ? pos - keys.low + keys.sinks + 1 : 0;
        const int sink_end = a.sinks < 0x7fffffffu ? (int)a.sinks : 0x7fffffff;
        int from = 0;
        if (a.window != 0 && pos >= 0 && (unsigned)pos >= a.window) from = pos - (int)a.window + 1 - keys.low + keys.sinks;
        const float sl2 = Cfg::F16 ? __fmul_rn(sl2_all, sh->row[0][r]) : sl2_all;
        const unsigned t_lane = taddr + ((unsigned)((warp & 3) * 32) << 16);
        float m = NO_MAX, l = 0.f;
        float acc[OC];
#pragma unroll
        for (int i = 0; i < OC; i++) acc[i] = 0.f;
        bool ok = true;
        auto wait = [&](uint64_t *bar, int phase) {  // a warp goes on together: TMEM accesses are warp-wide
            ok = __all_sync(0xffffffffu, ok && pr_wait(bar, (unsigned)phase & 1u, sh, kv));
        };
        // adds this half of tile j's w.v to the row's sums
        auto gather = [&](int j) {
            wait(&sh->o_full[j & 1], j >> 1);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < OC; c += 32) {
                float o[32];
                tmem_ld32(t_lane + Cfg::T_O + (j & 1) * HDP + x * OC + c, o);
                tmem_wait_ld();
                pin32(o);
#pragma unroll
                for (int i = 0; i < 32; i++) acc[c + i] = __fadd_rn(acc[c + i], o[i]);
            }
        };
        float v[CT];  // this thread's scores of a tile
        auto fetch = [&](int j) {
            wait(&sh->s_full[j & 1], j >> 1);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < CT; c += 32) tmem_ld32(t_lane + (j & 1) * Cfg::T_S + x * CT + c, v + c);
        };
        if (ntile > 0) fetch(0);
        for (int j = 0; j < ntile && ok; j++) {
            const unsigned t_s = t_lane + (j & 1) * Cfg::T_S;
            tmem_wait_ld();  // tile j's scores, on their way since the last tile's end
#pragma unroll
            for (int c = 0; c < CT; c += 32) pin32(v + c);
            const int i0 = lo + j * KT + x * CT;
            const unsigned *valid = &sh->valid[j & 7][x * CT / 32];
            bool whole = i0 + CT <= to && i0 + CT <= hi && (i0 + CT <= sink_end || i0 >= from);
#pragma unroll
            for (int c = 0; c < CT / 32; c++) whole = whole && valid[c] == 0xffffffffu;
            if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
                for (int g = 0; g < CT; g += 32) {
                    // bit c: list position i0 + g + c is seen
                    auto below = [&](int end) -> unsigned {
                        const int n = end - (i0 + g);
                        return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
                    };
                    const unsigned seen = below(to) & (below(sink_end) | ~below(from)) & valid[g >> 5];
#pragma unroll
                    for (int c = 0; c < 32; c++) v[g + c] = seen & (1u << c) ? v[g + c] : -INFINITY;
                }
            }
            float t0 = v[0], t1 = v[1], t2 = v[2], t3 = v[3];
#pragma unroll
            for (int c = 4; c < CT; c += 4) {
                t0 = fmaxf(t0, v[c]);
                t1 = fmaxf(t1, v[c + 1]);
                t2 = fmaxf(t2, v[c + 2]);
                t3 = fmaxf(t3, v[c + 3]);
            }
            const float top = __fmul_rn(fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)), sl2);
            // this thread has its scores, and says whether its row's reference
            // has to move; the first weights are worked out meanwhile, as if none had
            if (top > m + Range::rescale) *(volatile int *)&sh->move[j & 3] = 1;
            warp_arrive(&sh->seen_all);
            float sum;  // of 32 weights
            unsigned w[NQ][16];
            auto weights = [&](int c) {
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float e0 = exp2_approx(__fmaf_rn(v[c + i], sl2, -m)), e1 = exp2_approx(__fmaf_rn(v[c + i + 1], sl2, -m));
                    s0 = __fadd_rn(s0, e0);
                    s1 = __fadd_rn(s1, e1);
                    unsigned p[NQ];
                    split2_weights<TYPE, NQ>(e0, e1, p);
#pragma unroll
                    for (int n = 0; n < NQ; n++) w[n][i / 2] = p[n];
                }
                sum = __fadd_rn(s0, s1);
            };
            weights(0);
            wait(&sh->seen_all, j);
            if (!ok) break;
            float f = 1.0f;
            const bool moved = *(volatile int *)&sh->move[j & 3] != 0;
            if (tid == 0) *(volatile int *)&sh->move[(j + 2) & 3] = 0;  // last read two tiles ago
            if (moved) {  // the halves of each row move their reference together
                *(volatile float *)&sh->row[x][r] = top;
                warp_arrive(&sh->swapped);
                wait(&sh->swapped, 0);
                if (!ok) break;
                const float both = fmaxf(top, *(volatile float *)&sh->row[x ^ 1][r]);
                warp_arrive(&sh->swapped);
                wait(&sh->swapped, 1);  // read before the next exchange
                if (!ok) break;
                if (both > m + Range::rescale) {
                    const float to_m = __fsub_rn(both, Range::margin);
                    f = exp2_approx(__fsub_rn(m, to_m));
                    m = to_m;
                    l = __fmul_rn(l, f);
                }
                weights(0);
            }
            // every score of the tile is in registers: the weights take their place
#pragma unroll
            for (int c = 0; c < CT; c += 32) {
                if (c > 0) weights(c);
                l = __fadd_rn(l, sum);
#pragma unroll
                for (int n = 0; n < NQ; n++) tmem_st16(t_s + n * (KT / 2) + (x * CT + c) / 2, w[n]);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&sh->p_full[j & 1]);
            if (j + 1 < ntile) fetch(j + 1);
            if (j > 0 && ok) gather(j - 1);  // under w.v of this tile
            if (moved) {
#pragma unroll
                for (int i = 0; i < OC; i++) acc[i] = __fmul_rn(acc[i], f);
            }
        }
        if (ok && ntile > 0) gather(ntile - 1);
        // (a thread that broke off leaves the others' waits to give up: all meet here)
        const bool done = !named_bar_or(2, 256, !ok);
        sh->row[x][r] = l;
        named_bar_sync(2, 256);
        if (done) {
            l = __fadd_rn(sh->row[0][r], sh->row[1][r]);
            const bool whole = plan.splits == 1;
            const float inv = !whole ? 1.0f : l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
            // every product is complete: the results go through the q tiles,
            // 16-byte chunk c of row r at chunk c ^ (r & 7), to whole rows
            float4 *s_o = reinterpret_cast<float4 *>(s_q);
            // Once a reference was set, l is 2^margin or more, but for scores past
            // 2^24, of which x - m keeps the bits that m, rounded, has lost: they
            // may add up to any power of two, and the weights to zero or infinity.
            bool finite = fabsf(l) < INFINITY && (m == NO_MAX || l >= Range::least);
#pragma unroll
            for (int i = 0; i < OC; i += 4) {
                float y[4] = {acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    y[u] = __fmul_rn(y[u], inv);
                    if (x * OC + i < hd) finite = finite && fabsf(y[u]) < INFINITY;
                }
                s_o[r * (HDP / 4) + (((x * OC + i) / 4) ^ (r & 7))] = make_float4(y[0], y[1], y[2], y[3]);
            }
            if (!whole && x == 0 && row_ok)
                plan.part_ml[((size_t)row * a.num_heads + h) * plan.splits + split] = make_float2(m, l);
            named_bar_sync(2, 256);
            const bool vec = !whole || (((uintptr_t)a.out | (a.ldo * 4)) & 15) == 0;
            constexpr int LPR = HDP / 4, RPP = 32 / LPR;  // lanes a row, rows a pass
            const int c = lane % LPR;
            const unsigned my_flat = flat0 + (unsigned)(warp * 16 + (lane & 15)), my_tok = my_flat / (unsigned)group;
            const size_t my_row = (size_t)(row0 + (int)my_tok);
            const int my_head = head * group + (int)(my_flat - my_tok * (unsigned)group);
            const long long my_at = (int)my_tok >= rows ? -1
                                    : whole ? (long long)(my_row * a.ldo + (size_t)my_head * hd)
                                            : (long long)(((my_row * a.num_heads + my_head) * plan.splits + split) * hd);
            float *const to_base = (whole ? a.out : plan.part_o) + c * 4;
#pragma unroll 4
            for (int i = 0; i < 16; i += RPP) {
                const int rr = warp * 16 + i + lane / LPR;
                const long long at = __shfl_sync(0xffffffffu, my_at, i + lane / LPR);
                if (at < 0 || c * 4 >= hd) continue;
                float *dst = to_base + at;
                const float4 y = s_o[rr * LPR + (c ^ (rr & 7))];
                if (vec)
                    *reinterpret_cast<float4 *>(dst) = y;
                else
                    dst[0] = y.x, dst[1] = y.y, dst[2] = y.z, dst[3] = y.w;
            }
            // rows that met a value that is not finite, or scores so large, once their first
            // results are written (the barrier orders the stores)
            if (named_bar_or(2, 256, row_ok && !finite)) {
                sh->row[x][r] = finite ? 0.f : 1.f;
                named_bar_sync(2, 256);
                unsigned redo = __ballot_sync(0xffffffffu, x == 0 && row_ok && (sh->row[0][r] != 0.f || sh->row[1][r] != 0.f));
                while (redo) {
                    const int who = __ffs(redo) - 1;
                    redo &= redo - 1;
                    const int rrow = __shfl_sync(0xffffffffu, row, who), rh = __shfl_sync(0xffffffffu, h, who);
                    const int rfrom = __shfl_sync(0xffffffffu, from, who), rto = __shfl_sync(0xffffffffu, to, who);
                    const RowState st = attend_row<TYPE>(kv, b, seq, head, a.q + (size_t)rrow * a.ldq + (size_t)rh * hd,
                                                         sl2_all, keys, lo, hi, rfrom, sink_end, rto);
                    const size_t at = ((size_t)rrow * a.num_heads + rh) * plan.splits + split;
                    float *d = whole ? a.out + (size_t)rrow * a.ldo + (size_t)rh * hd : plan.part_o + at * hd;
                    const float div = whole ? st.l : 1.0f;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (lane + 32 * c < hd) d[lane + 32 * c] = div == 0.f ? 0.f : __fdiv_rn(st.acc[c], div);
                    if (!whole && lane == 0) plan.part_ml[at] = make_float2(st.m, st.l);
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
            constexpr unsigned idesc_s = umma_idesc_f16(TYPE != KV_F16, 128, KT, false);
            const unsigned idesc_o = umma_idesc_f16(TYPE != KV_F16, 128, (hd + 15) / 16 * 16, true);
            const unsigned a_q = smem_addr(pr_smem), a_kv = a_q + Cfg::QBYTES;
            bool ok = true;
            auto wait = [&](uint64_t *bar, int phase) {  // the warp goes on together
                ok = __all_sync(0xffffffffu, ok && pr_wait(bar, (unsigned)phase & 1u, sh, kv));
                tc_fence_after();
            };
            // the products of parts that count, the smallest first
            auto parts = [&](auto f) {
                if constexpr (NC == 1) {
#pragma unroll
                    for (int i = NQ - 1; i >= 0; i--) f(i, 0, i == NQ - 1);
                } else {
                    f(2, 0, true), f(0, 2, false), f(1, 1, false), f(1, 0, false), f(0, 1, false), f(0, 0, false);
                }
            };
            // tile j, of parity P: every operand is a constant
            auto scores = [&](auto parity, int j) {
                constexpr int P = decltype(parity)::value, S = Cfg::NSLOT == 4 ? 2 * P : 0;
                wait(&sh->full[S], Cfg::NSLOT == 4 ? j >> 1 : j);
                fence_async_elected();
                if (!ok) return;
                parts([&](int i, int c, bool first) {
#pragma unroll
                    for (int ks = 0; ks < HDP / 16; ks++) {
                        const unsigned ao = i * Cfg::QPART + (ks >> 2) * 128 * 128 + (ks & 3) * 32;
                        const unsigned bo = S * Cfg::SLOT + c * Cfg::PART + (ks >> 2) * KT * 128 + (ks & 3) * 32;
                        if (Cfg::F16 && i == 0 && ks == 0)
                            tc_mma_f16_onto_part2(P * Cfg::T_S, umma_desc_sw128(a_q + ao), umma_desc_sw128(a_kv + bo), idesc_s);
                        else
                            tc_mma_f16(P * Cfg::T_S, umma_desc_sw128(a_q + ao), umma_desc_sw128(a_kv + bo), idesc_s,
                                       !first || ks > 0);
                    }
                });
                tc_commit_elected(&sh->s_full[P]);
                tc_commit_elected(&sh->empty[S]);
            };
            auto values = [&](auto parity, int j) {
                constexpr int P = decltype(parity)::value, S = Cfg::NSLOT == 4 ? 2 * P + 1 : 1;
                wait(&sh->full[S], Cfg::NSLOT == 4 ? j >> 1 : j);
                fence_async_elected();
                wait(&sh->p_full[P], j >> 1);
                if (!ok) return;
                parts([&](int i, int c, bool first) {
#pragma unroll
                    for (int ks = 0; ks < KT / 16; ks++) {
                        const unsigned w_at = P * Cfg::T_S + i * (KT / 2) + ks * 8;
                        const uint64_t v_desc = umma_desc_sw128_mn(a_kv + S * Cfg::SLOT + c * Cfg::PART + ks * 2048, KT * 128);
                        if (Cfg::F16 && i == 0 && ks == 0)
                            tc_mma_f16_ta_onto_part2(Cfg::T_O + P * HDP, w_at, v_desc, idesc_o);
                        else
                            tc_mma_f16_ta(Cfg::T_O + P * HDP, w_at, v_desc, idesc_o, !first || ks > 0);
                    }
                });
                tc_commit_elected(&sh->o_full[P]);
                tc_commit_elected(&sh->empty[S]);
            };
            const std::integral_constant<int, 0> even{};
            const std::integral_constant<int, 1> odd{};
            wait(&sh->q_full, 0);
            scores(even, 0);
            // q.k of tile j + 1 goes over the weights of tile j - 1, which its
            // w.v has read by then
            for (int j = 0; j < ntile && ok; j += 2) {
                if (j + 1 < ntile) scores(odd, j + 1);
                values(even, j);
                if (j + 1 == ntile) break;
                if (j + 2 < ntile) scores(even, j + 2);
                values(odd, j + 1);
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
        constexpr int CH = HDP / 8;               // 16-byte chunks of a row's part
        constexpr int RSTEP = Cfg::PRODUCERS / CH;  // rows a pass: 12, 6, 28 or 14
        constexpr int PASSES = (KT + RSTEP - 1) / RSTEP;
        constexpr int ES = TYPE == KV_F32 ? 4 : 2;
        static_assert(Cfg::PRODUCERS % CH == 0, "a thread keeps its chunk");
        const int c = p % CH, r_first = p / CH;
        const bool in_row = c * 8 < hd;
        // the chunk's place in its row, swizzled, for the passes by four
        unsigned place[4];
#pragma unroll
        for (int n = 0; n < 4; n++) place[n] = sw16_off((r_first + n * RSTEP) & 7, c, KT) - ((r_first + n * RSTEP) & 7) * 128;
        int slot = 0;
        unsigned turn = 1;  // phase of an empty slot: none is waited for in the first round
        bool first_round = true;
        bool ok = true, all_held = false;
        // byte offset in the pools of key `i` of tile j, -1 for none
        auto find = [&](int j, int i) -> long long {
            const int at = lo + j * KT + i;
            const long long o = i < KT && at < hi ? key_offset(kv, b, seq, (unsigned)keys.key(at), head) : -1;
            return o < 0 ? -1 : o * ES;
        };
        long long next0 = find(0, p), next1 = KT > Cfg::PRODUCERS ? find(0, p + Cfg::PRODUCERS) : -1;
        auto put = [&](const void *pool) {
            const int s = slot;
            if (!first_round) ok = pr_wait(&sh->empty[s], turn, sh, kv);
            if (++slot == Cfg::NSLOT) slot = 0, turn ^= 1u, first_round = false;
            if (!ok) return;
            unsigned char *dst = s_kv + s * Cfg::SLOT;
            if constexpr (TYPE != KV_F32) {
                const unsigned d0 = smem_addr(dst) + r_first * 128;
                const char *base = reinterpret_cast<const char *>(pool) + c * 16;
                if (in_row && all_held) {
#pragma unroll
                    for (int n = 0; n < PASSES; n++)
                        if (n < PASSES - 1 || r_first + n * RSTEP < KT)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(d0 + n * RSTEP * 128 + place[n & 3]),
                                         "l"(base + sh->off[r_first + n * RSTEP]));
                } else {
#pragma unroll 4
                    for (int n = 0; n < PASSES; n++) {
                        if (r_first + n * RSTEP >= KT) break;
                        const long long o = sh->off[r_first + n * RSTEP];
                        const bool in = o >= 0 && in_row;
                        const char *src = in ? base + o : reinterpret_cast<const char *>(pool);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d0 + n * RSTEP * 128 + place[n & 3]),
                                     "l"(src), "r"(in ? 16u : 0u));
                    }
                }
                // arrives once this thread's copies are in; the MMA warp orders
                // them before its own accesses
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_addr(&sh->full[s])) : "memory");
            } else {
                float4 u[PASSES][2];
#pragma unroll
                for (int n = 0; n < PASSES; n++) {
                    const int r = r_first + n * RSTEP;
                    const long long o = r < KT ? sh->off[r] : -1;
                    if (o >= 0 && in_row) {
                        const float4 *src = reinterpret_cast<const float4 *>(reinterpret_cast<const char *>(pool) + o + c * 32);
                        u[n][0] = src[0];
                        u[n][1] = src[1];
                    } else {
                        u[n][0] = u[n][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
#pragma unroll
                for (int n = 0; n < PASSES; n++) {
                    const int r = r_first + n * RSTEP;
                    if (r >= KT) continue;
                    unsigned part[4][3];
                    split2<KV_BF16, 3>(u[n][0].x, u[n][0].y, part[0]);
                    split2<KV_BF16, 3>(u[n][0].z, u[n][0].w, part[1]);
                    split2<KV_BF16, 3>(u[n][1].x, u[n][1].y, part[2]);
                    split2<KV_BF16, 3>(u[n][1].z, u[n][1].w, part[3]);
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        *reinterpret_cast<uint4 *>(dst + i * Cfg::PART + r * 128 + place[n & 3]) =
                            make_uint4(part[0][i], part[1][i], part[2][i], part[3][i]);
                }
                fence_async_smem();
                mbar_arrive(&sh->full[s]);
            }
        };
        for (int j = 0; j < ntile && ok; j++) {
            // tile j's offsets for all, then those of the next tile on their way
            if (p < KT) sh->off[p] = next0;
            const unsigned held0 = __ballot_sync(0xffffffffu, next0 >= 0);
            if (lane == 0 && p < KT) sh->valid[j & 7][p >> 5] = held0;
            unsigned held1 = 0xffffffffu;
            if (KT > Cfg::PRODUCERS && warp == 9) {
                sh->off[Cfg::PRODUCERS + p] = next1;
                held1 = __ballot_sync(0xffffffffu, next1 >= 0);
                if (lane == 0) sh->valid[j & 7][3] = held1;
            }
            all_held = !named_bar_or(1, Cfg::PRODUCERS, (p < KT && held0 != 0xffffffffu) || held1 != 0xffffffffu);
            if (j + 1 < ntile) {
                next0 = find(j + 1, p);
                if (KT > Cfg::PRODUCERS && warp == 9) next1 = find(j + 1, p + Cfg::PRODUCERS);
            }
            if constexpr (TYPE == KV_F32) {  // one copy of the long conversion
#pragma unroll 1
                for (int i = 0; i < 2 && ok; i++) put(i == 0 ? kv.k : kv.v);
            } else {
                put(kv.k);
                if (ok) put(kv.v);
            }
            ok = !named_bar_or(1, Cfg::PRODUCERS, !ok);
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
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
    launch_kernel(paged_rows_kernel<TYPE, HDP>, dim3(grid), dim3(RowsCfg<TYPE, HDP>::THREADS), RowsCfg<TYPE, HDP>::SMEM, s, false, kv, b, a,
                  plan);
}

}  // namespace

RowsPlan plan_paged_rows(const KvView &kv, const BatchView &b, const PagedAttnView &a, uint32_t max_kv_len) {
    RowsPlan p{};
    const uint64_t group = a.num_heads / kv.kv_heads;
    const uint64_t rt = 128, kt = kv.type == KV_F16 ? 128 : 64;
    // a tile may end inside each sequence: an upper bound of their number
    p.tiles = (uint64_t)b.num_rows * group / rt + (uint64_t)std::min(b.num_seqs, b.num_rows);
    const uint64_t units = std::max<uint64_t>(p.tiles * kv.kv_heads, 1);
    uint64_t most = max_kv_len;
    if (a.window) most = std::min<uint64_t>(most, (uint64_t)a.window + a.sinks + rt / group + 1);
    const uint64_t key_tiles = (most + kt - 1) / kt;
    // fewer tiles than SMs: split the keys, at least four key tiles each
    const uint64_t splits = units < 148 ? std::min<uint64_t>(148 / units, key_tiles / 4) : 1;
    p.splits = (int)std::max<uint64_t>(splits, 1);
    const uint64_t rows = (uint64_t)b.num_rows * a.num_heads, parts = p.splits > 1 ? rows * p.splits : 0;
    p.ml_bytes = parts_ml_bytes(parts);
    // The bound for every call of as many rows and keys or fewer, which may be
    // split more: units tiles hold at most 128 x units (row, query head) pairs,
    // and units x splits is at most 148.
    const uint64_t more = std::min<uint64_t>(148, key_tiles / 4);
    const uint64_t bound = more > 1 ? std::min(rows * more, 148 * rt) : 0;
    p.scratch_bytes = parts_bytes(std::max(parts, bound), kv.hd);
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
