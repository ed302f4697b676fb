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

// a warp per row; shared memory: the row's ordered keys
__global__ void router_groups_kernel(const RouterArgs A) {
    extern __shared__ unsigned long long router_smem[];
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int row = blockIdx.x * warps + warp;
    if (row >= A.rows) return;  // whole warps leave together
    unsigned long long* key = router_smem + (size_t)warp * A.experts;
    const float* x = A.logits + (size_t)row * A.experts;

    float mx = -INFINITY;
    double inv = 1.0;
    if (!A.sigmoid) {
        for (int e = lane; e < A.experts; e += 32) mx = fmaxf(mx, x[e]);  // a NaN never wins
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    auto raw = [&](float v) -> double {  // the score before the division by the softmax sum; 0 for a closed expert
        if (v != v || v == -INFINITY) return 0.0;
        if (A.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
        return v == mx ? 1.0 : exp((double)v - (double)mx);
    };
    if (!A.sigmoid) {
        double sum = 0.0;
        for (int e = lane; e < A.experts; e += 32) sum += raw(x[e]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_d(sum, o);
        inv = sum > 0.0 ? sum : 1.0;
    }
    for (int e = lane; e < A.experts; e += 32) {
        const float v = x[e];
        const bool closed = v != v || v == -INFINITY;
        key[e] = closed ? kClosed : ordered(raw(v) / inv + (A.bias ? (double)A.bias[e] : 0.0));
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
        if (lane == s) sel_mine = bi, w_mine = raw(x[bi]) / inv;
        __syncwarp();
        if (lane == 0) key[bi] = kTaken;
        __syncwarp();
    }
    if (A.normalize) {
        double total = 0.0;
        for (int s = 0; s < A.k; ++s) total += __shfl_sync(0xffffffffu, w_mine, s);
        if (total > 0.0) w_mine /= total;
    }
    if (lane < A.k) {
        A.selected[(size_t)row * A.k + lane] = sel_mine;
        A.weights[(size_t)row * A.k + lane] = (float)(w_mine * (double)A.scale);
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
    const RouterArgs a{logits_dev, bias_dev, (int)seq, (int)n_expert, (int)top_k, score == FQ_SCORE_SIGMOID, (int)n_group, (int)topk_group,
                       group_score == FQ_GROUP_TOP2, normalize != 0, scale, selected_dev, weights_dev};
    const int warps = n_expert <= 1024 ? 4 : 1;  // eight bytes of shared memory per expert and warp, 32 KB at most
    const cudaError_t e = launch_pdl(router_groups_kernel, dim3((unsigned)((seq + warps - 1) / warps)), dim3(warps * 32),
                                     sizeof(unsigned long long) * n_expert * warps, st, a);
    g_trace.launches++;
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "router launch");
}
