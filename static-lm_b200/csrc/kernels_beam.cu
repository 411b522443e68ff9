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

constexpr int BS_THREADS = 256, BS_WARPS = BS_THREADS / 32;
constexpr int BS_PER = 16, BS_CHUNK = BS_THREADS * BS_PER;  // logits of a thread, and of a CTA, at a time
constexpr int BS_MAX_OUT = 64;

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

// CTA (row, part).  The list of the part's best so far has a threshold, its
// num_out-th: most chunks hold no logit above it, and cost a maximum, an exp and
// a vote.  Where more pass than the buffer takes (the first chunk, rising
// logits), the num_out-th largest of the threads' own maxima is a bound below
// which nothing can be among the best, and at most 16 num_out pass that.
template <bool VEC>
__global__ void __launch_bounds__(BS_THREADS) beam_part_kernel(BeamView a, BeamPlan plan) {
    __shared__ uint64_t s_cand[17 * BS_MAX_OUT], s_best[BS_MAX_OUT], s_top[BS_THREADS];
    __shared__ int s_count[BS_WARPS];
    __shared__ float s_m[BS_WARPS];
    __shared__ double s_s[BS_WARPS];
    pdl_release();
    const int row = blockIdx.x / plan.parts, part = blockIdx.x % plan.parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.num_out, cap = 17 * K;
    if (!row_lives(a, row)) return;  // the join knows
    const int begin = part * plan.part, end = min(a.vocab, begin + plan.part);
    const float *x = a.logits + (size_t)row * a.ld;
    auto token = [&](int at, int i) { return VEC ? at + (i >> 2) * (4 * BS_THREADS) + tid * 4 + (i & 3) : at + i * BS_THREADS + tid; };
    auto load = [&](int at, float (&v)[BS_PER]) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < BS_PER; i += 4) {
                const int t = token(at, i);
                float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (t + 3 < end) {
                    f = *reinterpret_cast<const float4 *>(x + t);
                } else if (t < end) {
                    f.x = x[t];
                    if (t + 1 < end) f.y = x[t + 1];
                    if (t + 2 < end) f.z = x[t + 2];
                }
                v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < BS_PER; i++) {
                const int t = token(at, i);
                v[i] = t < end ? x[t] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < BS_PER; i++) v[i] = fmaxf(v[i], -INFINITY);  // NaN is no candidate and adds nothing
    };
    float m = -INFINITY, s = 0.f, least = -INFINITY;  // least: of the list, once it is full
    int held = 0;
    for (int at = begin; at < end; at += BS_CHUNK) {
        float v[BS_PER];
        load(at, v);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < BS_PER; i++) top = fmaxf(top, v[i]);
        if (top > m) {
            s = __fmul_rn(s, exp2_approx(__fmul_rn(__fsub_rn(m, top), 1.44269504088896340736f)));
            m = top;
        }
        if (m > -INFINITY) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int i = 0; i < BS_PER; i += 2) {
                s0 = __fadd_rn(s0, exp2_approx(__fmul_rn(__fsub_rn(v[i], m), 1.44269504088896340736f)));
                s1 = __fadd_rn(s1, exp2_approx(__fmul_rn(__fsub_rn(v[i + 1], m), 1.44269504088896340736f)));
            }
            s = __fadd_rn(s, __fadd_rn(s0, s1));
        }
        if (!__syncthreads_or(top > least)) continue;
        uint64_t bound = 0;
        int mine = 0, base = 0, total = 0;
        auto count = [&]() {  // of this thread's that pass, its place among all, and all
            mine = 0;
#pragma unroll
            for (int i = 0; i < BS_PER; i++) mine += v[i] > least && beam_key(v[i], token(at, i)) >= bound;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += t;
            }
            if (lane == 31) s_count[warp] = sum;
            __syncthreads();
            base = sum - mine;
            total = 0;
#pragma unroll
            for (int w = 0; w < BS_WARPS; w++) {
                if (w < warp) base += s_count[w];
                total += s_count[w];
            }
        };
        count();
        if (held + total > cap) {
            float best = v[0];
            int which = 0;
#pragma unroll
            for (int i = 1; i < BS_PER; i++)
                if (v[i] > best) best = v[i], which = i;
            s_top[tid] = best > least ? beam_key(best, token(at, which)) : 0;
            __syncthreads();
            if (warp == 0) {
                uint64_t t[BS_WARPS], one = 0;
#pragma unroll
                for (int i = 0; i < BS_WARPS; i++) t[i] = s_top[i * 32 + lane];
                for (int k = 0; k < K; k++) {
                    uint64_t mx = 0;
#pragma unroll
                    for (int i = 0; i < BS_WARPS; i++) mx = t[i] > mx ? t[i] : mx;
                    one = warp_max64(mx);
#pragma unroll
                    for (int i = 0; i < BS_WARPS; i++) t[i] = t[i] == one ? 0 : t[i];
                }
                if (lane == 0) s_top[0] = one;
            }
            __syncthreads();
            bound = s_top[0];
            count();
        }
        int place = held + base;
#pragma unroll
        for (int i = 0; i < BS_PER; i++) {
            if (mine && v[i] > least) {
                const uint64_t key = beam_key(v[i], token(at, i));
                if (key >= bound) s_cand[place++] = key;
            }
        }
        held += total;
        __syncthreads();
        if (held > K) {  // every candidate's rank; the first K stay, in order
            for (int e = tid; e < held; e += BS_THREADS) {
                const uint64_t key = s_cand[e];
                int rank = 0;
                for (int o = 0; o < held; o++) rank += s_cand[o] > key;
                if (rank < K) s_best[rank] = key;
            }
            __syncthreads();
            if (tid < K) s_cand[tid] = s_best[tid];
            held = K;
            least = key_logit(s_best[K - 1]);
            __syncthreads();
        } else if (held == K) {
            uint64_t low = s_cand[0];
            for (int o = 1; o < held; o++) low = s_cand[o] < low ? s_cand[o] : low;
            least = key_logit(low);
        }
    }
    // the list, sorted, and the part's maximum and sum
    float all = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    if (lane == 0) s_m[warp] = all;
    __syncthreads();
    all = s_m[0];
#pragma unroll
    for (int w = 1; w < BS_WARPS; w++) all = fmaxf(all, s_m[w]);
    double sum = m > -INFINITY ? (double)__fmul_rn(s, exp2_approx(__fmul_rn(__fsub_rn(m, all), 1.44269504088896340736f))) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_s[warp] = sum;
    __syncthreads();
    const size_t list = (size_t)row * plan.parts + part;
    if (tid == 0) {
        sum = 0.0;
        for (int w = 0; w < BS_WARPS; w++) sum += s_s[w];
        plan.part_ms[list] = make_double2((double)all, sum);
    }
    uint64_t *best = plan.part_best + list * K;
    for (int e = tid; e < K; e += BS_THREADS) {
        if (e < held) {
            const uint64_t key = s_cand[e];
            int rank = 0;
            for (int o = 0; o < held; o++) rank += s_cand[o] > key;
            best[rank] = key;
        } else {
            best[e] = 0;  // no token
        }
    }
}

// One group: the sums of its rows, then num_out times the best head of its
// rows' lists.
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

__global__ void __launch_bounds__(BS_THREADS) beam_join_kernel(BeamView a, BeamPlan plan) {
    extern __shared__ double s_lse[];  // [beams]: log sum exp; NaN for a row without candidates
    __shared__ uint64_t s_head[2][BS_WARPS];
    __shared__ int s_list[2][BS_WARPS];
    double *const s_score = s_lse + a.beams;
    unsigned char *const s_next = reinterpret_cast<unsigned char *>(s_score + a.beams);  // [list]: places taken
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int row0 = blockIdx.x * a.beams, lists = a.beams * plan.parts, K = a.num_out;
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
    for (int i = tid; i < lists; i += blockDim.x) s_next[i] = 0;
    __syncthreads();
    // the candidate at a list's head, 0 for none
    auto head = [&](int list, int &tok) -> uint64_t {
        const int beam = list / plan.parts, at = s_next[list];
        const double lse = s_lse[beam];
        if (lse != lse || at >= K) return 0;
        if (a.ended && a.ended[row0 + beam] != 0) {
            tok = a.end_token;
            return list % plan.parts == 0 && at == 0 ? ordered64(s_score[beam]) : 0;
        }
        const uint64_t key = plan.part_best[((size_t)row0 * plan.parts + list) * K + at];
        tok = key_token(key);
        return key ? ordered64(s_score[beam] + ((double)key_logit(key) - lse)) : 0;
    };
    uint64_t best = 0;
    int from = 0, tok = 0;
    auto refresh = [&]() {
        best = 0;
        for (int i = tid; i < lists; i += blockDim.x) {
            int t;
            const uint64_t h = head(i, t);
            if (h > best) best = h, from = i, tok = t;
        }
    };
    refresh();
    for (int k = 0; k < K; k++) {
        const uint64_t w = warp_max64(best);
        const int list = (int)__reduce_min_sync(0xffffffffu, best == w && w ? (unsigned)from : 0x7fffffffu);
        if (lane == 0) s_head[k & 1][warp] = w, s_list[k & 1][warp] = list;
        __syncthreads();
        uint64_t win = 0;
        int which = 0x7fffffff;
        for (int i = 0; i < warps; i++) {
            const uint64_t h = s_head[k & 1][i];
            const int li = s_list[k & 1][i];
            if (h > win || (h == win && li < which)) win = h, which = li;
        }
        const size_t to = (size_t)blockIdx.x * K + k;
        if (win == 0) {
            if (tid == 0) a.out_scores[to] = -INFINITY, a.out_rows[to] = a.out_tokens[to] = -1;
        } else if (best == win && from == which) {
            const uint64_t u = win >> 63 ? win & ~(1ull << 63) : ~win;
            a.out_scores[to] = (float)__longlong_as_double((long long)u);
            a.out_rows[to] = row0 + which / plan.parts;
            a.out_tokens[to] = tok;
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
    // parts enough to fill the GPU, at most 64
    constexpr uint64_t CTAS = 148 * 6;
    const uint64_t most = std::min<uint64_t>(chunks, 64);
    const uint64_t want = std::max<uint64_t>(std::min<uint64_t>((CTAS + rows - 1) / std::max<uint64_t>(rows, 1), most), 1);
    const uint64_t per = (chunks + want - 1) / want;
    p.part = (int)std::min<uint64_t>(per * BS_CHUNK, INT32_MAX / 2 + 1);
    p.parts = (int)((chunks + per - 1) / per);
    // no fewer for fewer rows or tokens: rows x parts is below rows + CTAS and at most rows x most
    const uint64_t lists = std::min(rows * most, rows + CTAS);
    p.scratch_bytes = lists * (sizeof(double2) + 8ull * a.num_out);
    return p;
}

void launch_beam_select(const BeamView &a, const BeamPlan &plan, cudaStream_t s) {
    const unsigned grid = (unsigned)((uint64_t)a.groups * a.beams * plan.parts);
    if (a.vec)
        launch_kernel(beam_part_kernel<true>, dim3(grid), dim3(BS_THREADS), 0, s, false, a, plan);
    else
        launch_kernel(beam_part_kernel<false>, dim3(grid), dim3(BS_THREADS), 0, s, false, a, plan);
    const int lists = a.beams * plan.parts, warps = std::min((lists + 31) / 32, BS_WARPS);
    launch_kernel(beam_join_kernel, dim3((unsigned)a.groups), dim3((unsigned)warps * 32), (size_t)a.beams * 16 + lists, s, true, a,
                  plan);
}

}  // namespace slm
