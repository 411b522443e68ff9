// kernels_beam.cu -- beam search: the best continuations of each group of beams
// over the vocabulary.
//
// A candidate is score_b + x_bv - log sum_u exp x_bu.  Within a row the order
// is that of the logits, so one pass over a row's part keeps its largest
// num_out logits and (m, s) with s = sum exp(x - m); two such pairs join as
// m = max, s = sum of s_i exp(m_i - m).  A second launch forms the sums of a
// group's rows in 64 bits and merges their parts' sorted lists.
#include "async.cuh"
#include "kernels.h"

namespace slm {

namespace {

constexpr int BS_MAX_OUT = 64;
constexpr int BS_THREADS = 128, BS_WARPS = BS_THREADS / 32;
constexpr int BS_STAGES = 3, BS_PER = 16, BS_CHUNK = 32 * BS_PER;  // logits of a lane, and of a warp, at a time
constexpr int BJ_THREADS = 256, BJ_WARPS = BJ_THREADS / 32, BS_MAX_PARTS = 128;

// Logit and token as one number: larger for a larger logit, and for the lower
// token of two that are equal.  Zeros of either sign are equal.
__device__ __forceinline__ uint64_t beam_key(float x, int token) {
    unsigned u = __float_as_uint(__fadd_rn(x, 0.0f));
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)u << 32 | (0xffffffffu - (unsigned)token);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const unsigned u = (unsigned)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_token(uint64_t key) { return (int)(0xffffffffu - (unsigned)key); }

// The largest of a warp's numbers.
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ bool row_lives(const BeamView &a, int row) {
    return fabsf(a.scores[row]) < INFINITY && !(a.ended && a.ended[row] != 0);
}

// CTA (row, part); its warps take chunks of 512 logits in turn, each through its
// own ring of cp.async stages.  A chunk costs a maximum, an exp and a vote unless a
// logit passes the CTA's threshold, a key that num_out of its logits are known to lie
// above: those that do go one by one into the warp's best so far, a list over its
// lanes, rank r in lane r (and r - 32), by a count of the ranks above and a shift.
// The threshold is first a bound from the warps' first chunks, by the lanes' own
// largest: num_out of one chunk reach it.  From then on each warp publishes its
// ceil(num_out / 4)-th best (s_place): the four warps hold num_out between them that
// are no lower than the least of the four, which goes into s_least by an atomic
// maximum, as does the last place of a warp's own full list.  Both only rise, so one
// that is read late is a lower threshold that holds too.  Where more than a few of
// a chunk pass (rising logits), the chunk's own bound comes first: at most 16
// num_out are not below that.  No warp waits for another but after the first chunk
// and before the lists are merged.
// 256 rows of 131072 (134 MB, 20.5 us), both launches, 44.3 us; one list a CTA, with a
// barrier a chunk, 85; a list a warp without a common threshold 63; loads to registers
// instead of the rings 55.
template <bool VEC, bool TWO>
__global__ void __launch_bounds__(BS_THREADS, 8) beam_part_kernel(BeamView a, BeamPlan plan) {
    extern __shared__ __align__(16) float s_ring[];  // [warp][stage][512]
    __shared__ uint64_t s_best[BS_WARPS * BS_MAX_OUT];
    __shared__ unsigned long long s_least;
    __shared__ volatile uint64_t s_place[BS_WARPS];  // the warps' r-th best
    __shared__ float s_m[BS_WARPS];
    __shared__ double s_s[BS_WARPS];
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = a.num_out;
    const int row = (int)(blockIdx.x / (unsigned)plan.parts), part = (int)(blockIdx.x % (unsigned)plan.parts);
    if (!row_lives(a, row)) return;  // the join knows
    const int begin = part * plan.part, end = min(a.vocab, begin + plan.part);
    const float *x = a.logits + (size_t)row * a.ld;
    float *const ring = s_ring + warp * (BS_STAGES * BS_CHUNK);
    // element i of this lane in a chunk
    auto place = [&](int i, int l) { return (i >> 2) * 128 + l * 4 + (i & 3); };
    auto fetch = [&](int at, int stage) {
        const unsigned dst = smem_addr(ring + stage * BS_CHUNK);
        if (at < end) {
            if constexpr (VEC) {  // (rows are multiples of 16 bytes apart: what is past the row's end is not read)
#pragma unroll
                for (int i = 0; i < BS_PER; i += 4) {
                    const int o = place(i, lane), n = min(max(end - at - o, 0), 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst + o * 4), "l"(x + (n ? at + o : 0)), "r"(n * 4));
                }
            } else {
#pragma unroll
                for (int i = 0; i < BS_PER; i++) {
                    const int o = i * 32 + lane;
                    const bool in = at + o < end;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst + o * 4), "l"(x + (in ? at + o : 0)),
                                 "r"(in ? 4u : 0u));
                }
            }
        }
        cp_async_commit();
    };
    auto load = [&](int at, int stage, float (&v)[BS_PER]) {
        const unsigned src = smem_addr(ring + stage * BS_CHUNK);
#pragma unroll
        for (int i = 0; i < BS_PER; i += 4) {
            const float4 f = lds_f32x4(src + place(i, lane) * 4);
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
        if (at + BS_CHUNK > end) {
#pragma unroll
            for (int i = 0; i < BS_PER; i++) v[i] = at + place(i, lane) < end ? v[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < BS_PER; i++) v[i] = fmaxf(v[i], -INFINITY);  // NaN is no candidate and adds nothing
    };
    constexpr int STEP = BS_WARPS * BS_CHUNK;
    const int first = begin + warp * BS_CHUNK;
#pragma unroll
    for (int i = 0; i < BS_STAGES - 1; i++) fetch(first + i * STEP, i);
    const int r = (K + BS_WARPS - 1) / BS_WARPS - 1;  // (below 16)
    if (threadIdx.x < BS_WARPS) s_place[threadIdx.x] = 0;
    if (threadIdx.x == 0) s_least = 0;
    __syncthreads();
    float m = -INFINITY;
    double s = 0.0;           // this lane's sum of exp(x - m): in f32 its error grows with the row's length
    uint64_t low = 0;         // the threshold as this warp last saw it; 0: none
    float least = -FLT_MAX;   // its logit (-infinity is no candidate)
    auto see = [&](uint64_t key) {
        if (key > low) low = key, least = key_logit(key);
    };
    uint64_t k0 = 0, k1 = 0;  // ranks lane and 32 + lane; 0: none
    auto last = [&]() -> uint64_t { return __shfl_sync(0xffffffffu, TWO && K > 32 ? k1 : k0, (K - 1) & 31); };
    auto insert = [&](uint64_t key) {
        const int above = __popc(__ballot_sync(0xffffffffu, k0 > key));
        const uint64_t up = __shfl_up_sync(0xffffffffu, k0, 1);
        if constexpr (TWO) {
            const int above1 = above + __popc(__ballot_sync(0xffffffffu, k1 > key));
            uint64_t up1 = __shfl_up_sync(0xffffffffu, k1, 1);
            const uint64_t carry = __shfl_sync(0xffffffffu, k0, 31);
            if (lane == 0) up1 = carry;
            if (lane + 32 > above1) k1 = up1;
            if (lane + 32 == above1) k1 = key;
        }
        if (lane > above) k0 = up;
        if (lane == above) k0 = key;
    };
    int stage = 0;
    for (int at = first; at < end || at == first; at += STEP) {
        cp_async_wait<BS_STAGES - 2>();
        __syncwarp();
        float v[BS_PER];
        load(at, stage, v);
        const int here = stage * BS_CHUNK;
        fetch(at + (BS_STAGES - 1) * STEP, stage == 0 ? BS_STAGES - 1 : stage - 1);
        stage = stage == BS_STAGES - 1 ? 0 : stage + 1;
        float top = v[0];
#pragma unroll
        for (int i = 1; i < BS_PER; i++) top = fmaxf(top, v[i]);
        if (at == first) {
            // a first threshold: num_out lanes' largest reach it (up to 32), or all lanes' second largest
            float bound;
            if (TWO && K > 32) {
                float two = -INFINITY, one = v[0];
#pragma unroll
                for (int i = 1; i < BS_PER; i++) two = fmaxf(two, fminf(one, v[i])), one = fmaxf(one, v[i]);
                bound = -warp_max_nan(-two);
            } else {
                float rest = top;
                int n = 0;
                do {
                    bound = warp_max_nan(rest);
                    n += __popc(__ballot_sync(0xffffffffu, rest == bound));
                    if (rest == bound) rest = -INFINITY;
                } while (n < K && bound > -INFINITY);
            }
            if (lane == 0 && bound > -INFINITY) atomicMax(&s_least, (unsigned long long)(beam_key(bound, 0) | 0xffffffffu) - 0xffffffffull - 1);
            __syncthreads();
        }
        // (as lane 0 read it: other warps write it meanwhile, and the lanes go on together only
        // where low is the same in all of them)
        see(__shfl_sync(0xffffffffu, *(volatile unsigned long long *)&s_least, 0));
        if (top > m) {
            s *= (double)exp2_approx(__fmul_rn(__fsub_rn(m, top), 1.44269504088896340736f));
            m = top;
        }
        if (m > -INFINITY) {
            const uint64_t minus_m = pack2(-m, -m), log2e = pack2(1.44269504088896340736f, 1.44269504088896340736f);
            uint64_t sums = 0;
#pragma unroll
            for (int i = 0; i < BS_PER; i += 2) {
                float e0, e1;
                unpack2(mul2(add2(pack2(v[i], v[i + 1]), minus_m), log2e), e0, e1);
                sums = add2(sums, pack2(exp2_approx(e0), exp2_approx(e1)));
            }
            float s0, s1;
            unpack2(sums, s0, s1);
            s += (double)__fadd_rn(s0, s1);
        }
        if (!__any_sync(0xffffffffu, top >= least)) continue;
        unsigned pass = 0;  // of this lane's
#pragma unroll
        for (int i = 0; i < BS_PER; i++) pass |= (unsigned)(v[i] >= least) << i;
        if (__reduce_add_sync(0xffffffffu, __popc(pass)) > 32u) {
            uint64_t one = 0, two = 0;
#pragma unroll
            for (int i = 0; i < BS_PER; i++) {
                const uint64_t key = pass >> i & 1u ? beam_key(v[i], at + place(i, lane)) : 0;
                if (key > one)
                    two = one, one = key;
                else if (TWO && key > two)
                    two = key;
            }
            uint64_t bound = 0;
            if (TWO && K > 32) {
                bound = ~warp_max64(~two);
            } else {
                for (int k = 0; k < K; k++) {
                    bound = warp_max64(one);
                    if (one == bound) one = 0;
                }
            }
            if (bound) see(bound - 1);
            pass = 0;
#pragma unroll
            for (int i = 0; i < BS_PER; i++) pass |= (unsigned)(v[i] >= least && beam_key(v[i], at + place(i, lane)) > low) << i;
        }
        for (unsigned lanes = __ballot_sync(0xffffffffu, pass); lanes; lanes &= lanes - 1) {
            const int l = __ffs(lanes) - 1;
            for (unsigned its = __shfl_sync(0xffffffffu, pass, l); its; its &= its - 1) {
                const int o = place(__ffs(its) - 1, l);
                const uint64_t key = beam_key(ring[here + o], at + o);
                if (key <= low) continue;
                insert(key);
                see(last());
            }
        }
        // (places only rise: one that is read late is a lower bound too)
        const uint64_t mine = __shfl_sync(0xffffffffu, k0, r);
        if (lane == 0) s_place[warp] = mine;
        const uint64_t all = ~warp_max64(lane < BS_WARPS ? ~(lane == warp ? mine : s_place[lane]) : 0);
        if (all) see(all - 1);
        if (lane == 0 && low > *(volatile unsigned long long *)&s_least) atomicMax(&s_least, (unsigned long long)low);
    }
    cp_async_wait<0>();
    // the warps' lists become one
    if (lane < K) s_best[warp * K + lane] = k0;
    if (TWO && lane + 32 < K) s_best[warp * K + lane + 32] = k1;
    const size_t list = (size_t)row * plan.parts + part;
    float all = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    double sum = m > -INFINITY ? s * (double)exp2_approx(__fmul_rn(__fsub_rn(m, all), 1.44269504088896340736f)) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_m[warp] = all, s_s[warp] = sum;
    __syncthreads();
    if (threadIdx.x == BS_THREADS - 1) {
        all = s_m[0];
        for (int w = 1; w < BS_WARPS; w++) all = fmaxf(all, s_m[w]);
        sum = 0.0;
        for (int w = 0; w < BS_WARPS; w++)
            if (s_m[w] > -INFINITY) sum += s_s[w] * exp((double)s_m[w] - (double)all);
        plan.part_ms[list] = make_double2((double)all, sum);
    }
    uint64_t *best = plan.part_best + list * K;
    const int held = BS_WARPS * K;
    for (int e0 = 0; e0 < held; e0 += BS_THREADS / 4) {  // an entry's rank, by four lanes; among those that are none, by place
        const int e = e0 + threadIdx.x / 4;
        const uint64_t key = e < held ? s_best[e] : 0;
        int rank = 0;
        for (int o = threadIdx.x & 3; o < held; o += 4) rank += s_best[o] > key || (key == 0 && s_best[o] == 0 && o < e);
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (e < held && (threadIdx.x & 3) == 0 && rank < K) best[rank] = key;
    }
}

// One group: the sums of its rows, then num_out times the best head of its
// rows' lists.
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(BeamView a, BeamPlan plan, int staged) {
    extern __shared__ double s_lse[];  // [beams]: log sum exp; NaN for a row without candidates
    // staged: entries of all lists, where they are in shared memory
    __shared__ uint64_t s_head[2][BJ_WARPS], s_key[2][BJ_WARPS];
    __shared__ int s_list[2][BJ_WARPS];
    double *const s_score = s_lse + a.beams;
    uint64_t *const s_keys = reinterpret_cast<uint64_t *>(s_score + a.beams), *const s_cand = s_keys + staged;
    unsigned char *const s_next = reinterpret_cast<unsigned char *>(s_cand + staged);  // [list]: places taken
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int row0 = blockIdx.x * a.beams, lists = a.beams * plan.parts, K = a.num_out;
    for (int i = tid; i < lists; i += blockDim.x) s_next[i] = 0;
    pdl_wait();
    for (int i = warp; i < a.beams; i += warps) {
        const int row = row0 + i;
        const bool ended = a.ended && a.ended[row] != 0;
        const float score = a.scores[row];
        double lse = 0.0;
        if (!(fabsf(score) < INFINITY)) {
            lse = __longlong_as_double(0x7ff8000000000000ll);
        } else if (!ended) {
            double m = -INFINITY, s = 0.0;
            for (int j = lane; j < plan.parts; j += 32) m = fmax(m, plan.part_ms[(size_t)row * plan.parts + j].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int j = lane; j < plan.parts; j += 32) {
                const double2 p = plan.part_ms[(size_t)row * plan.parts + j];
                if (p.y > 0.0) s += p.y * exp(p.x - m);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            lse = m + log(s);
            if (!(fabs(lse) < INFINITY)) lse = __longlong_as_double(0x7ff8000000000000ll);
        }
        if (lane == 0) s_lse[i] = lse, s_score[i] = (double)score;
    }
    const uint64_t *const keys = plan.part_best + (size_t)row0 * plan.parts * K;
    for (int i = tid; i < staged; i += blockDim.x) s_keys[i] = keys[i];
    __syncthreads();
    // the candidate at a list's head, 0 for none
    auto head = [&](int list, uint64_t &key) -> uint64_t {
        const int beam = list / plan.parts, at = s_next[list];
        const double lse = s_lse[beam];
        if (lse != lse || at >= K) return 0;
        if (a.ended && a.ended[row0 + beam] != 0) {
            key = beam_key(0.f, a.end_token);
            return list % plan.parts == 0 && at == 0 ? ordered64(s_score[beam]) : 0;
        }
        key = keys[(size_t)list * K + at];
        return key ? ordered64(s_score[beam] + ((double)key_logit(key) - lse)) : 0;
    };
    auto put = [&](int k, uint64_t win, int list, int token) {
        const size_t to = (size_t)blockIdx.x * K + k;
        const uint64_t u = win >> 63 ? win & ~(1ull << 63) : ~win;
        a.out_scores[to] = win ? (float)__longlong_as_double((long long)u) : -INFINITY;
        a.out_rows[to] = win ? row0 + list / plan.parts : -1;
        a.out_tokens[to] = win ? token : -1;
    };
    // Of equal sums that of the lower row is first, then that of its larger logit and lower
    // token: the larger key, which may be in any of the row's lists.
    auto first = [&](bool &mine, int list, uint64_t key) {
        const unsigned those = __ballot_sync(0xffffffffu, mine);
        if (those & (those - 1)) {
            const unsigned beam = (unsigned)(list / plan.parts);
            const unsigned lowest = __reduce_min_sync(0xffffffffu, mine ? beam : 0xffffffffu);
            mine = mine && beam == lowest;
            const uint64_t largest = warp_max64(mine ? key : 0);
            mine = mine && key == largest;
        }
    };
    if (staged) {
        // every entry's sum at once; then a warp with up to four lists a lane picks,
        // without barriers.  (Sums worked out as heads come up: four rows of 49152 15.2 us
        // instead of 12.5.)
        for (int i = tid; i < staged; i += blockDim.x) {
            const int list = i / K, at = i - list * K, beam = list / plan.parts;
            const double lse = s_lse[beam];
            const uint64_t key = s_keys[i];
            uint64_t cand = key ? ordered64(s_score[beam] + ((double)key_logit(key) - lse)) : 0;
            if (a.ended && a.ended[row0 + beam] != 0)
                cand = list % plan.parts == 0 && at == 0 ? ordered64(s_score[beam]) : 0;
            s_cand[i] = lse == lse ? cand : 0;
        }
        __syncthreads();
        if (warp > 0) return;
        uint64_t h[4];
        int at[4] = {0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 4; u++) h[u] = lane + 32 * u < lists ? s_cand[(lane + 32 * u) * K] : 0;
        for (int k = 0; k < K; k++) {
            uint64_t best = h[0];
            int from = 0;
#pragma unroll
            for (int u = 1; u < 4; u++)
                if (h[u] > best) best = h[u], from = u;
            const uint64_t win = warp_max64(best);
            if (win == 0) {
                if (lane == 0) put(k, 0, 0, 0);
                continue;
            }
            bool mine = best == win, twice = false;
#pragma unroll
            for (int u = 1; u < 4; u++) twice = twice || (h[u] == win && from < u);
            const unsigned those = __ballot_sync(0xffffffffu, mine), more = __ballot_sync(0xffffffffu, twice);
            if ((those & (those - 1)) | more) {
                uint64_t key = 0;
                int beam = -1;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    if (h[u] != win) continue;
                    const int list = lane + 32 * u, its = list / plan.parts;
                    const uint64_t its_key = s_keys[list * K + at[u]];
                    if (beam < 0 || (its == beam && its_key > key)) beam = its, key = its_key, from = u;
                }
                first(mine, lane + 32 * from, key);
            }
            if (mine) {
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (from == u) {
                        const int list = lane + 32 * u, i = list * K + at[u];
                        const bool ended = a.ended && a.ended[row0 + list / plan.parts] != 0;
                        put(k, win, list, ended ? a.end_token : key_token(s_keys[i]));
                        h[u] = ++at[u] < K ? s_cand[i + 1] : 0;
                    }
            }
        }
        return;
    }
    const int pickers = (int)blockDim.x;
    uint64_t best = 0, its = 0;  // a sum and its key
    int from = 0;
    auto refresh = [&]() {
        best = 0;
        for (int i = tid; i < lists; i += pickers) {
            uint64_t key;
            const uint64_t h = head(i, key);
            if (h > best || (h == best && h && i / plan.parts == from / plan.parts && key > its)) best = h, from = i, its = key;
        }
    };
    refresh();
    for (int k = 0; k < K; k++) {
        uint64_t win = warp_max64(best);
        bool mine = best == win && win;
        first(mine, from, its);
        if (mine || (win == 0 && lane == 0)) s_head[k & 1][warp] = win, s_list[k & 1][warp] = from, s_key[k & 1][warp] = its;
        __syncthreads();
        int which = 0x7fffffff;
        uint64_t key = 0;
        win = 0;
        for (int i = 0; i < warps; i++) {
            const uint64_t h = s_head[k & 1][i], hk = s_key[k & 1][i];
            const int li = s_list[k & 1][i], d = li / plan.parts - which / plan.parts;
            if (h > win || (h == win && h && (d < 0 || (d == 0 && hk > key)))) win = h, which = li, key = hk;
        }
        if (win == 0) {
            if (tid == 0) put(k, 0, 0, 0);
        } else if (best == win && from == which) {
            put(k, win, which, key_token(key));
            s_next[which]++;
            refresh();
        }
    }
}

}  // namespace

BeamPlan plan_beam_select(const BeamView &a) {
    BeamPlan p{};
    const uint64_t rows = (uint64_t)a.groups * a.beams;
    const uint64_t chunks = std::max<uint64_t>(((uint64_t)a.vocab + BS_CHUNK - 1) / BS_CHUNK, 1);
    // Parts of at least a chunk for every warp, the number with the least work by
    // this count: of the SM with the most CTAs the rounds of chunks, and for each
    // CTA about four more for its start and end; fewer than four CTAs an SM leave
    // the memory idle.  (256 rows of 131072, 1, 2, 3, 4, 5, 6, 8 parts: 57, 50.7,
    // 50.2, 48.2, 54.4, 54.5, 56.5 us; four of 49152, 2, 4, 6, 8, 12: 19.5, 17.2,
    // 16.1, 16.1, 16.3.)
    constexpr uint64_t SMS = 148, MOST = 32 * SMS;  // CTAs where rows are split
    const uint64_t most = std::max<uint64_t>(std::min<uint64_t>(chunks / BS_WARPS, BS_MAX_PARTS), 1);
    uint64_t best = UINT64_MAX;
    for (uint64_t n = 1; n <= most && (n == 1 || rows * n <= MOST); n++) {
        const uint64_t per = (chunks + n - 1) / n, parts = (chunks + per - 1) / per;
        const uint64_t cost = std::max<uint64_t>((rows * parts + SMS - 1) / SMS, 4) * ((per + BS_WARPS - 1) / BS_WARPS + 4);
        if (cost >= best) continue;
        best = cost;
        p.part = (int)std::min<uint64_t>(per * BS_CHUNK, INT32_MAX / 2 + 1);
        p.parts = (int)parts;
    }
    // no fewer for fewer rows or tokens
    const uint64_t lists = std::max(rows, std::min(rows * most, MOST));
    p.scratch_bytes = lists * (sizeof(double2) + 8ull * a.num_out);
    return p;
}

void launch_beam_select(const BeamView &a, const BeamPlan &plan, cudaStream_t s) {
    const dim3 grid((unsigned)((uint64_t)a.groups * a.beams * plan.parts)), block(BS_THREADS);
    auto go = [&](auto *kernel, SmemOptIn &opt) {
        constexpr int bytes = BS_WARPS * BS_STAGES * BS_CHUNK * 4;
        opt(kernel, bytes);
        // (its CTAs come while the kernel before ends, and wait: 46.7 to 44.3 us, 12.3 to 10.0)
        launch_kernel(kernel, grid, block, bytes, s, true, a, plan);
    };
    static SmemOptIn opt[4];
    if (a.num_out <= 32)
        a.vec ? go(beam_part_kernel<true, false>, opt[0]) : go(beam_part_kernel<false, false>, opt[1]);
    else
        a.vec ? go(beam_part_kernel<true, true>, opt[2]) : go(beam_part_kernel<false, true>, opt[3]);
    const int lists = a.beams * plan.parts, warps = std::min(std::max((lists + 31) / 32, a.beams), BJ_WARPS);
    // (at most 4 KB of sums, 32 KB of lists and a byte for each of 32 * 148: rows are cut into no more parts in all)
    const int staged = lists <= 128 && lists * a.num_out <= 2048 ? lists * a.num_out : 0;
    launch_kernel(beam_join_kernel, dim3((unsigned)a.groups), dim3((unsigned)warps * 32), (size_t)a.beams * 16 + staged * 16 + lists,
                  s, true, a, plan, staged);
}

}  // namespace slm
