// Expert router with softmax or sigmoid scores, a balance bias and expert groups.
//
//   score_e = sigmoid(x_e)  or  exp(x_e - max x) / sum exp(x - max x)
//   key_e   = score_e + bias_e                    (chooses, never weighs)
//   rank_g  = max of the group's keys, or the sum of its two largest
//   chosen  = the top_k largest keys among the topk_group groups of largest rank
//   w_e     = score_e [/ sum of the chosen scores] * scale
//
// The softmax top-k without bias or groups is the reference's router (src/exec/topk.zig:21-86, router_topk_kernel); this
// one serves the layers that balance their experts by a bias. Keys are 64-bit: among 256 experts two keys lie within
// f32 rounding of each other about once in ten thousand tokens, and a router that then picks by rounding does not
// reproduce.
//
// Bound: latency for a token, instruction issue for a batch (the logits are 4 bytes per 30 instructions). So a row is first
// ranked on f32 keys whose error has a bound, in registers, a contiguous run of experts per lane; where the ranks'
// neighbours lie further apart than twice the bound the 64-bit order is the same, and 64-bit arithmetic is needed for the
// chosen scores alone. Otherwise (a few rows in a thousand, and ties) the row is ranked again on 64-bit keys. Rows of
// more than 512 experts or 32 groups are ranked on 64-bit keys in shared memory at once.
//
// Measured (B200): 4099 tokens over 256 experts, sigmoid, bias, four of eight groups: 37 us with 64-bit keys for every row, 15
// us in this form, of which a row in doubt takes some 4 (the last of them ends the kernel); one token over 128 experts 5.2 us,
// the launch.
#include "internal.h"
#include "runtime.h"

namespace fq {

namespace {

constexpr int kMaxExperts = 4096;
constexpr int kMaxChosen = 32;
constexpr int kMaxGroups = 64;

struct RouterArgs {
    const float* logits;
    const float* bias;
    int rows, experts, k, sigmoid, groups, kept, top2, normalize;
    int lanes;  // of a group, a power of two (see Place)
    float scale;
    int* selected;
    float* weights;
};

// Keys as unsigned integers in key order: 0 a taken entry, 1 a closed one (-infinity), larger numbers open experts.
constexpr unsigned long long kTaken = 0, kClosed = 1;
__device__ __forceinline__ unsigned long long ordered(double key) {
    const long long b = __double_as_longlong(key + 0.0);  // -0 and +0 are one key
    if (key != key || b == (long long)0xfff0000000000000ull) return kClosed;
    return (unsigned long long)b ^ (b < 0 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double key_of(unsigned long long u) {
    if (u <= kClosed) return -INFINITY;
    return __longlong_as_double((long long)(u ^ (u >> 63 ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ double shfl_xor_d(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// the largest (value, lowest index) over the warp
__device__ __forceinline__ void warp_best(unsigned long long& v, int& i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
    }
}

// A row's 64-bit scores: what a warp needs to turn a logit into one.
struct Scores {
    bool sigmoid;
    float mx;      // softmax: the largest logit
    double total;  // softmax: the sum of exp(x - mx)
    // before the division by the softmax sum; 0 for a closed expert
    __device__ __forceinline__ double raw(float v) const {
        if (v != v || v == -INFINITY) return 0.0;
        if (sigmoid) return 1.0 / (1.0 + exp(-(double)v));
        return v == mx ? 1.0 : exp((double)v - (double)mx);
    }
};

// The largest logit and, for a softmax, the 64-bit sum.
__device__ __forceinline__ Scores row_scores(const RouterArgs& A, const float* x, int lane) {
    Scores r{A.sigmoid != 0, -INFINITY, 1.0};
    if (A.sigmoid) return r;
    for (int e = lane; e < A.experts; e += 32) r.mx = fmaxf(r.mx, x[e]);  // a NaN never wins
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.mx = fmaxf(r.mx, __shfl_xor_sync(0xffffffffu, r.mx, o));
    double sum = 0.0;
    for (int e = lane; e < A.experts; e += 32) sum += r.raw(x[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_d(sum, o);
    r.total = sum > 0.0 ? sum : 1.0;
    return r;
}

// Weights of the chosen experts (lane s holds slot s and its score) and the row's results.
__device__ __forceinline__ void write_row(const RouterArgs& A, int row, int lane, int sel, double w) {
    if (A.normalize) {
        double total = 0.0;
        for (int s = 0; s < A.k; ++s) total += __shfl_sync(0xffffffffu, w, s);
        if (total > 0.0) w /= total;
    }
    if (lane < A.k) {
        A.selected[(size_t)row * A.k + lane] = sel;
        A.weights[(size_t)row * A.k + lane] = (float)(w * (double)A.scale);
    }
}

// A row ranked on 64-bit keys, held in shared memory.
__device__ __noinline__ void route_row_exact(const RouterArgs A, int row, int lane, unsigned long long* key) {
    const float* x = A.logits + (size_t)row * A.experts;
    const Scores sc = row_scores(A, x, lane);
    for (int e = lane; e < A.experts; e += 32) {
        const float v = x[e];
        const bool closed = v != v || v == -INFINITY;
        key[e] = closed ? kClosed : ordered(sc.raw(v) / sc.total + (A.bias ? (double)A.bias[e] : 0.0));
    }
    __syncwarp();
    if (A.groups > 1) {
        const int size = A.experts / A.groups;
        unsigned long long rank[kMaxGroups / 32];
#pragma unroll
        for (int t = 0; t < kMaxGroups / 32; ++t) {
            const int g = lane + 32 * t;
            rank[t] = kTaken;
            if (g < A.groups) {
                unsigned long long a = 0, b = 0;  // the two largest
                for (int i = 0; i < size; ++i) {
                    const unsigned long long u = key[g * size + i];
                    if (u > a) b = a, a = u;
                    else if (u > b) b = u;
                }
                rank[t] = A.top2 && size > 1 ? ordered(key_of(a) + key_of(b)) : a;
            }
        }
        unsigned long long open = 0;
        for (int r = 0; r < A.kept; ++r) {
            unsigned long long v = rank[0];
            int i = v == kTaken ? 0x7fffffff : lane;
#pragma unroll
            for (int t = 1; t < kMaxGroups / 32; ++t)
                if (rank[t] > v) v = rank[t], i = lane + 32 * t;
            warp_best(v, i);
            open |= 1ull << i;
#pragma unroll
            for (int t = 0; t < kMaxGroups / 32; ++t)
                if (i == lane + 32 * t) rank[t] = kTaken;
        }
        for (int e = lane; e < A.experts; e += 32)
            if (!((open >> (e / size)) & 1)) key[e] = kClosed;
        __syncwarp();
    }

    double w_mine = 0.0;  // lane s keeps slot s
    int sel_mine = 0;
    for (int s = 0; s < A.k; ++s) {
        unsigned long long bv = kTaken;
        int bi = 0x7fffffff;
        for (int e = lane; e < A.experts; e += 32)
            if (key[e] > bv) bv = key[e], bi = e;
        warp_best(bv, bi);
        if (lane == s) sel_mine = bi, w_mine = sc.raw(x[bi]) / sc.total;
        __syncwarp();
        if (lane == 0) key[bi] = kTaken;
        __syncwarp();
    }
    write_row(A, row, lane, sel_mine, w_mine);
}

// Which experts a lane holds: each group on `lanes` lanes of its own, NE consecutive experts a lane, in order. A group's last
// lanes may be partly or wholly empty.
template <int NE>
struct Place {
    int first, count;  // experts first .. first + count - 1
    bool leader;       // the group's first lane
    __device__ __forceinline__ Place(const RouterArgs& A, int lane) {
        const int size = A.experts / A.groups, group = lane / A.lanes, at = (lane - group * A.lanes) * NE;
        first = group * size + at;
        count = group < A.groups ? max(0, min(NE, size - at)) : 0;
        leader = group < A.groups && at == 0;
    }
};

// The lane that holds the warp's largest value (0: none), the lowest of several: by the upper halves, then the lower ones.
__device__ __forceinline__ int best_lane(unsigned long long mine) {
    const unsigned hi = (unsigned)(mine >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    unsigned who = __ballot_sync(0xffffffffu, hi == top);
    if (who & (who - 1)) {
        const unsigned lo = hi == top ? (unsigned)mine : 0u, top_lo = __reduce_max_sync(0xffffffffu, lo);
        who = __ballot_sync(0xffffffffu, hi == top && lo == top_lo);
    }
    return __ffs(who) - 1;
}

// A row ranked on 64-bit keys, NE experts per lane, in registers.
template <int NE>
__device__ __noinline__ void route_row_exact(const RouterArgs A, int row, int lane) {
    const float* x = A.logits + (size_t)row * A.experts;
    Scores sc{A.sigmoid != 0, -INFINITY, 1.0};
    const Place<NE> mine(A, lane);
    float v[NE];
    double p[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) v[j] = j < mine.count ? x[mine.first + j] : -INFINITY;
    if (!A.sigmoid) {
#pragma unroll
        for (int j = 0; j < NE; ++j) sc.mx = fmaxf(sc.mx, v[j]);  // a NaN never wins
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sc.mx = fmaxf(sc.mx, __shfl_xor_sync(0xffffffffu, sc.mx, o));
    }
#pragma unroll
    for (int j = 0; j < NE; ++j) p[j] = sc.raw(v[j]);
    if (!A.sigmoid) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NE; ++j) sum += p[j];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_d(sum, o);
        sc.total = sum > 0.0 ? sum : 1.0;
    }
    unsigned long long key[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) {
        if (!A.sigmoid) p[j] /= sc.total;
        const bool closed = !(v[j] > -INFINITY);
        key[j] = j >= mine.count ? kTaken : closed ? kClosed : ordered(p[j] + (A.bias ? (double)A.bias[mine.first + j] : 0.0));
    }
    if (A.groups > 1) {
        const int size = A.experts / A.groups, lanes = A.lanes;
        unsigned long long a = 0, b = 0;  // the two largest of the lane, then of the group's lanes
#pragma unroll
        for (int j = 0; j < NE; ++j) {
            if (key[j] > a) b = a, a = key[j];
            else if (key[j] > b) b = key[j];
        }
        for (int o = 1; o < lanes; o <<= 1) {
            const unsigned long long oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
            const unsigned long long low = a < oa ? a : oa, second = b > ob ? b : ob;
            b = low > second ? low : second, a = a > oa ? a : oa;
        }
        unsigned long long rank = !mine.leader ? kTaken : A.top2 && size > 1 ? ordered(key_of(a) + key_of(b)) : a;
        unsigned open = 0;
        for (int r = 0; r < A.kept; ++r) {
            const int who = best_lane(rank);
            open |= (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << who;
            if (lane == who) rank = kTaken;
        }
        if (!((open >> lane) & 1)) {
#pragma unroll
            for (int j = 0; j < NE; ++j)
                if (key[j] != kTaken) key[j] = kClosed;
        }
    }
    double w_mine = 0.0;
    int sel_mine = 0;
    for (int s = 0; s < A.k; ++s) {
        unsigned long long top = key[0];
        int at = 0;
        double pv = p[0];
#pragma unroll
        for (int j = 1; j < NE; ++j)
            if (key[j] > top) top = key[j], at = j, pv = p[j];
        const int who = best_lane(top);
        const int e = __shfl_sync(0xffffffffu, mine.first + at, who);
        pv = __shfl_sync(0xffffffffu, pv, who);
        if (lane == s) sel_mine = e, w_mine = pv;
        if (lane == who) {
#pragma unroll
            for (int j = 0; j < NE; ++j)
                if (j == at) key[j] = kTaken;
        }
    }
    write_row(A, row, lane, sel_mine, w_mine);
}

// f32 keys as unsigned integers in key order; 0: taken or closed
__device__ __forceinline__ unsigned ordered32(float key) {
    const unsigned b = __float_as_uint(key + 0.0f);
    return b ^ ((int)b < 0 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float key_of32(unsigned u) { return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : ~0u)); }

// One round of a ranking over the warp's values, one per lane (0: none): the lane that holds the largest, or -1 where doubt
// remains: it is less than `apart` below the one before, or two lanes hold it, or it is no number. -2: none is left.
__device__ __forceinline__ int next_best(unsigned mine, float apart, float& prev) {
    const unsigned top = __reduce_max_sync(0xffffffffu, mine);
    if (top == 0) return -2;
    const float v = key_of32(top);
    const unsigned who = __ballot_sync(0xffffffffu, mine == top);
    if (!(prev - v > apart) || (who & (who - 1)) || !(fabsf(v) < INFINITY)) return -1;
    prev = v;
    return __ffs(who) - 1;
}

// Up to NE experts per lane (NE = 0: every row on 64-bit keys in shared memory). A warp per row.
template <int NE>
__global__ void __launch_bounds__(128) router_groups_kernel(const __grid_constant__ RouterArgs A) {
    extern __shared__ unsigned long long router_smem[];
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int row = blockIdx.x * warps + warp;
    if (row >= A.rows) return;  // whole warps leave together
    if constexpr (NE == 0) {
        route_row_exact(A, row, lane, router_smem + (size_t)warp * A.experts);
    } else {
        const float* x = A.logits + (size_t)row * A.experts;
        const Place<NE> mine(A, lane);
        float v[NE];
#pragma unroll
        for (int j = 0; j < NE; ++j) v[j] = j < mine.count ? x[mine.first + j] : -INFINITY;
        unsigned key[NE];
        float apart, mx = 0.0f;
        bool sure = true;
        const bool sums = A.groups > 1 && A.top2 && A.experts > A.groups;  // ranks add two keys
        // keys and twice the bound of their error. sigmoid: exp2 and the reciprocal are off by some 2^-22 each, the product in the
        // exponent by |x| 2^-23 where the score falls as e^-|x|: below 2^-20 together, the addition of the bias by 2^-24 of the key.
        // softmax without a bias: the logits themselves, exact; what lies e^-700 below the largest, or 1e-9 from a neighbour, is
        // left to 64 bits, where such scores may coincide. softmax with a bias, or where scores are added: below 4e-6 (exp2 2^-22,
        // the exponent's rounding |x - max| 2^-23 e^-|x - max|, at most 21 additions of the sum 2^-24 each, the division).
        if (A.sigmoid) {
            float big = 0.0f;
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const bool closed = !(v[j] > -INFINITY);  // NaN too
                const float s = __fdividef(1.0f, 1.0f + __expf(-fmaxf(v[j], -80.0f)));
                const float k = A.bias && j < mine.count ? s + A.bias[mine.first + j] : s;
                key[j] = closed ? 0u : ordered32(k);
                if (!closed) big = fmaxf(big, fabsf(k));
            }
            big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
            apart = 2.0f * (9.6e-7f + big * 1.2e-7f);
        } else {
            mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NE; ++j) mx = fmaxf(mx, v[j]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (A.bias || sums) {
                float p[NE], sum = 0.0f, big = 0.0f;
#pragma unroll
                for (int j = 0; j < NE; ++j) p[j] = v[j] > -INFINITY ? __expf(v[j] - mx) : 0.0f, sum += p[j];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float inv = 1.0f / sum;
#pragma unroll
                for (int j = 0; j < NE; ++j) {
                    const float k = A.bias && j < mine.count ? p[j] * inv + A.bias[mine.first + j] : p[j] * inv;
                    key[j] = v[j] > -INFINITY ? ordered32(k) : 0u;
                    if (v[j] > -INFINITY) big = fmaxf(big, fabsf(k));
                }
                big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
                apart = 2.0f * (4e-6f + big * 1.2e-7f);
            } else {
#pragma unroll
                for (int j = 0; j < NE; ++j) key[j] = v[j] > -INFINITY && v[j] - mx > -700.0f ? ordered32(v[j]) : 0u;
                apart = 1e-9f;
            }
        }
        if (A.groups > 1) {
            // the two best of the lane, then of the group's lanes; ranks of closed groups stay in doubt
            const int lanes = A.lanes;
            float a = -INFINITY, b = -INFINITY;
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const float k = key[j] ? key_of32(key[j]) : -INFINITY;
                if (k > a) b = a, a = k;
                else if (k > b) b = k;
            }
            for (int o = 1; o < lanes; o <<= 1) {
                const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
                b = fmaxf(fminf(a, oa), fmaxf(b, ob)), a = fmaxf(a, oa);
            }
            const float rank = sums ? a + b : a;
            unsigned rank_mine = mine.leader && rank > -INFINITY ? ordered32(rank) : 0u;
            unsigned open = 0;  // lanes of open groups
            const float far = rank_mine && sums ? 2.0f * apart + 2.4e-7f * (fabsf(a) + fabsf(b)) : apart;
            const float apart_ranks = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(far)));
            float prev = INFINITY;
            for (int r = 0; r < A.kept + (A.kept < A.groups); ++r) {
                const int who = next_best(rank_mine, apart_ranks, prev);
                if (who < 0) {
                    sure = sure && who == -2 && r == A.kept;
                    break;
                }
                if (r < A.kept) {
                    open |= (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << who;
                    if (lane == who) rank_mine = 0u;
                }
            }
            if (!((open >> lane) & 1)) {
#pragma unroll
                for (int j = 0; j < NE; ++j) key[j] = 0u;
            }
        }
        int sel_mine = 0;
        float v_mine = 0.0f;
        if (sure) {
            float prev = INFINITY;
            for (int r = 0; r <= A.k; ++r) {  // the first one not taken included
                unsigned top = key[0];
                int at = 0;
                float xv = v[0];
#pragma unroll
                for (int j = 1; j < NE; ++j)
                    if (key[j] > top) top = key[j], at = j, xv = v[j];
                // equal keys inside a lane: the second one shows in the next round, no distance apart
                const int who = next_best(top, apart, prev);
                if (who < 0) {
                    sure = who == -2 && r == A.k;
                    break;
                }
                const int e = __shfl_sync(0xffffffffu, mine.first + at, who);
                xv = __shfl_sync(0xffffffffu, xv, who);
                if (lane == r && r < A.k) sel_mine = e, v_mine = xv;
                if (lane == who) {
#pragma unroll
                    for (int j = 0; j < NE; ++j)
                        if (j == at) key[j] = 0u;
                }
            }
        }
        if (!sure) {
            route_row_exact<NE>(A, row, lane);
            return;
        }
        Scores sc{A.sigmoid != 0, mx, 1.0};
        if (!A.sigmoid && !A.normalize) sc = row_scores(A, x, lane);  // normalised weights do not need the sum of all
        write_row(A, row, lane, sel_mine, lane < A.k ? sc.raw(v_mine) / sc.total : 0.0);
    }
}

}  // namespace
}  // namespace fq

using namespace fq;

extern "C" int fq_router_groups_dev(const float* logits_dev, size_t seq, size_t n_expert, int score, const float* bias_dev, size_t n_group,
                                    size_t topk_group, int group_score, size_t top_k, int normalize, float scale, int32_t* selected_dev,
                                    float* weights_dev, void* stream) {
    if (!logits_dev || !selected_dev || !weights_dev) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (score != FQ_SCORE_SOFTMAX && score != FQ_SCORE_SIGMOID) return fail(FQ_DECLINED_ARGS, "score %d is not served", score);
    if (group_score != FQ_GROUP_MAX && group_score != FQ_GROUP_TOP2) return fail(FQ_DECLINED_ARGS, "group score %d is not served", group_score);
    if (seq == 0 || seq > (size_t)INT32_MAX) return fail(FQ_DECLINED_ARGS, "seq out of range");
    if (n_expert == 0 || n_expert > (size_t)kMaxExperts) return fail(FQ_DECLINED_ARGS, "n_expert=%zu: 1 to %d", n_expert, kMaxExperts);
    if (n_group == 0 || n_group > (size_t)kMaxGroups || n_expert % n_group != 0 || topk_group == 0 || topk_group > n_group)
        return fail(FQ_DECLINED_ARGS, "%zu of %zu groups over %zu experts", topk_group, n_group, n_expert);
    if (top_k == 0 || top_k > (size_t)kMaxChosen || top_k > topk_group * (n_expert / n_group)) return fail(FQ_DECLINED_ARGS, "bad top_k");
    if (!gpu_enabled()) return fail(FQ_DECLINED_GATE, "disabled by FUCINA_GPU=0");
    Ctx* ctx = context();
    if (!ctx) return FQ_DECLINED_NO_GPU;
    std::lock_guard<std::recursive_mutex> g(g_dispatch_lock);
    g_trace.calls++;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    RouterArgs a{logits_dev, bias_dev, (int)seq, (int)n_expert, (int)top_k, score == FQ_SCORE_SIGMOID, (int)n_group, (int)topk_group,
                       group_score == FQ_GROUP_TOP2, normalize != 0, 32, scale, selected_dev, weights_dev};
    const int warps = n_expert <= 1024 ? 4 : 1;  // eight bytes of shared memory per expert and warp, 32 KB at most
    const dim3 grid((unsigned)((seq + warps - 1) / warps)), block(warps * 32);
    // experts per lane: the fewest with which every group has 2^n lanes of its own
    auto fits = [&](size_t ne) {
        const size_t size = n_expert / n_group;
        a.lanes = 1;
        while (a.lanes * ne < size) a.lanes *= 2;
        return a.lanes * n_group <= 32;
    };
    cudaError_t e;
    if (fits(2)) e = launch_pdl(router_groups_kernel<2>, grid, block, 0, st, a);
    else if (fits(4)) e = launch_pdl(router_groups_kernel<4>, grid, block, 0, st, a);
    else if (fits(8)) e = launch_pdl(router_groups_kernel<8>, grid, block, 0, st, a);
    else if (fits(16)) e = launch_pdl(router_groups_kernel<16>, grid, block, 0, st, a);
    else e = launch_pdl(router_groups_kernel<0>, grid, block, sizeof(unsigned long long) * n_expert * warps, st, a);
    g_trace.launches++;
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "router launch");
}
