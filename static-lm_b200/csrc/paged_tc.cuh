// paged_tc.cuh -- what the tcgen05 kernels of the paged cache share: 16-bit
// operands in shared memory and TMEM, their MMAs, and TMEM <-> registers.
#pragma once

#include "async.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace slm {

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
// ---- the same of 16 columns, loaded, and 8, stored
__device__ __forceinline__ void tmem_ld16(unsigned taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pin16(float *v) {
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ void tmem_st8(unsigned taddr, const unsigned *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Rows that no sequence owns, shared out over the grid.
__device__ __forceinline__ void zero_unowned_rows(const KvView &kv, const BatchView &b, const PagedAttnView &a, int threads) {
    const int start = min(max(b.row_start[0], 0), b.num_rows);
    const int end = min(max(b.row_start[b.num_seqs], start), b.num_rows);
    for (long long i = blockIdx.x; i < (long long)b.num_rows - end + start; i += gridDim.x) {
        const long long r = i < start ? i : i - start + end;
        for (int e = threadIdx.x; e < a.num_heads * kv.hd; e += threads) a.out[(size_t)r * a.ldo + e] = 0.f;
    }
}

// Row tile `index` of (2^LOG2 rows each, the query heads of a KV head side by
// side), counted from the last sequence's last to the first, by one warp: its
// sequence's rows into sh->seq, row0, rows and past, its place among that
// sequence's tiles into sh->tile; sh->found whether there is one, sh->bits what
// row_start has wrong.
template <int LOG2, typename Shared>
__device__ __forceinline__ void find_row_tile(const BatchView &b, int group, int index, Shared *sh) {
    const int lane = threadIdx.x & 31;
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
        const int n = (int)(((long long)rows * group + (1 << LOG2) - 1) >> LOG2);
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

// One arrival for a warp's 32 threads (an arrival of each is worked off one by
// one: at 256 a tile they took longer than the arithmetic).
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

}  // namespace slm
