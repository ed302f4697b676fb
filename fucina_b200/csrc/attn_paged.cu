// Attention of one new token per sequence over a paged key-value cache.
//
//   out[s][h] = sum_j softmax_j(scale * q[s][h] . k[j]) v[j],   j in [max(0, len - window), len)
//
// with the running maximum m and sum l of the softmax: a key with score x changes (m, l, o) into
// (m', l e^(m - m') + e^(x - m'), o e^(m - m') + e^(x - m') v), m' = max(m, x), so K and V are read once. Two partial
// results over disjoint keys join the same way.
#include <cuda_fp16.h>

#include "internal.h"
#include "kvpages.h"
#include "runtime.h"

namespace fq {

namespace {

constexpr float kNegBig = -3.4e38f;
constexpr int kWarps = 4;

struct PagedArgs {
    KvView c;
    const float* q;
    size_t q_stride;
    const int* table;
    const int* len;
    int n_seqs, max_pages, max_len, heads, group;
    float scale;
    int window;
    float* out;
    float* stats;
    int* status;
};

// The keys sequence s sees; a length the call does not allow is cut and reported.
__device__ __forceinline__ void key_range(const PagedArgs& A, int s, int& first, int& end) {
    end = A.len[s];
    if (end < 0 || end > A.max_len) {
        *(volatile int*)A.status = FQ_ERR_PAGE;
        end = end < 0 ? 0 : A.max_len;
    }
    first = (A.window > 0 && end > A.window) ? end - A.window : 0;
}

// grid (heads, n_seqs): warp w takes the keys first + w, first + w + 4, ...; a lane holds the dims lane, lane + 32, ...
template <bool Q8>
__global__ void __launch_bounds__(kWarps * 32) attn_paged_kernel(const PagedArgs A) {
    __shared__ float sh_o[kWarps][kKvMaxD], sh_m[kWarps], sh_l[kWarps];
    pdl_wait_then_release();
    constexpr int ND = kKvMaxD / 32;
    const int h = blockIdx.x, s = blockIdx.y, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int d = A.c.d, kvh = h / A.group;
    int first, end;
    key_range(A, s, first, end);
    const float* qrow = A.q + (size_t)s * A.q_stride + (size_t)h * d;
    float q[ND], o[ND], m = kNegBig, l = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) q[t] = lane + 32 * t < d ? qrow[lane + 32 * t] : 0.0f, o[t] = 0.0f;
    for (int j = first + w; j < end; j += kWarps) {
        const KvSlot at = kv_slot(A.table, A.n_seqs, A.max_pages, A.c.page_tokens, A.c.n_pages, s, j);
        if (at.page < 0) {
            *(volatile int*)A.status = FQ_ERR_PAGE;
            continue;
        }
        const size_t row = (size_t)kvh * A.c.page_tokens + at.slot;
        const size_t e = (size_t)at.page * A.c.page_stride + row * d, sc = (size_t)at.page * A.c.scale_stride + row * (d >> 5);
        float x = 0.0f, v[ND];
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            const int i = lane + 32 * t;
            v[t] = 0.0f;
            if (i < d) {
                float k;
                if (Q8) {
                    k = (float)((const int8_t*)A.c.k)[e + i] * __half2float(A.c.k_scale[sc + t]);
                    v[t] = (float)((const int8_t*)A.c.v)[e + i] * __half2float(A.c.v_scale[sc + t]);
                } else {
                    k = __half2float(((const __half*)A.c.k)[e + i]);
                    v[t] = __half2float(((const __half*)A.c.v)[e + i]);
                }
                x = fmaf(q[t], k, x);
            }
        }
        x = group_sum<32>(x) * A.scale;
        const float m_new = fmaxf(m, x), r = expf(m - m_new), p = expf(x - m_new);
        l = l * r + p;
#pragma unroll
        for (int t = 0; t < ND; ++t) o[t] = fmaf(p, v[t], o[t] * r);
        m = m_new;
    }
#pragma unroll
    for (int t = 0; t < ND; ++t) sh_o[w][lane + 32 * t] = o[t];
    if (lane == 0) sh_m[w] = m, sh_l[w] = l;
    __syncthreads();
    float mm = kNegBig, ll = 0.0f;
    for (int i = 0; i < kWarps; ++i) mm = fmaxf(mm, sh_m[i]);
    for (int i = 0; i < kWarps; ++i) ll += sh_l[i] * expf(sh_m[i] - mm);
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        float a = 0.0f;
        for (int x = 0; x < kWarps; ++x) a += sh_o[x][i] * expf(sh_m[x] - mm);
        A.out[((size_t)s * A.heads + h) * d + i] = ll > 0.0f ? a / ll : 0.0f;
    }
    if (A.stats && threadIdx.x == 0) A.stats[((size_t)s * A.heads + h) * 2] = mm, A.stats[((size_t)s * A.heads + h) * 2 + 1] = ll;
}

}  // namespace
}  // namespace fq

using namespace fq;

extern "C" {

size_t fq_attn_paged_workspace_bytes(const fq_kv_pages* pages, size_t n_seqs, size_t heads, size_t max_len) {
    (void)pages, (void)n_seqs, (void)heads, (void)max_len;
    return 0;
}

int fq_attn_paged_dev(const fq_kv_pages* pages, const float* q_dev, size_t q_stride, const int32_t* page_table_dev, const int32_t* kv_len_dev,
                      size_t n_seqs, size_t max_pages, size_t max_len, size_t heads, float scale, size_t window, float* out_dev,
                      float* stats_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    (void)workspace_dev, (void)workspace_bytes;
    KvView c;
    if (int rc = check_kv_pages(pages, &c)) return rc;
    if (!q_dev || !page_table_dev || !kv_len_dev || !out_dev) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (heads == 0 || heads > 4096 || heads % c.kv_heads != 0) return fail(FQ_DECLINED_ARGS, "heads=%zu: a multiple of kv_heads=%d, at most 4096", heads, c.kv_heads);
    if (n_seqs == 0 || n_seqs > 65535) return fail(FQ_DECLINED_ARGS, "n_seqs=%zu: 1 to 65535", n_seqs);
    if (max_pages == 0 || max_pages > (size_t)INT32_MAX / c.page_tokens) return fail(FQ_DECLINED_ARGS, "max_pages=%zu out of range", max_pages);
    const size_t capacity = max_pages * c.page_tokens;
    if (max_len == 0 || max_len > capacity) max_len = capacity;
    if (q_stride == 0) q_stride = heads * c.d;
    if (q_stride < heads * c.d || q_stride % 4 != 0 || q_stride > ((size_t)1 << 32)) return fail(FQ_DECLINED_ARGS, "q_stride=%zu: at least heads * d and a multiple of 4", q_stride);
    if (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) return fail(FQ_DECLINED_ARGS, "q and out must be 16-byte aligned");
    if (!gpu_enabled()) return fail(FQ_DECLINED_GATE, "disabled by FUCINA_GPU=0");
    Ctx* ctx = context();
    if (!ctx) return FQ_DECLINED_NO_GPU;
    std::lock_guard<std::recursive_mutex> g(g_dispatch_lock);
    g_trace.calls++;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    if (window > max_len) window = 0;  // it covers every length
    PagedArgs a{c, q_dev, q_stride, page_table_dev, kv_len_dev, (int)n_seqs, (int)max_pages, (int)max_len, (int)heads, (int)(heads / c.kv_heads),
                scale, (int)window, out_dev, stats_dev, ctx->status_dev};
    const dim3 grid((unsigned)heads, (unsigned)n_seqs);
    const cudaError_t e = pages->fmt == FQ_KV_Q8_0 ? launch_pdl(attn_paged_kernel<true>, grid, dim3(kWarps * 32), 0, st, a)
                                                   : launch_pdl(attn_paged_kernel<false>, grid, dim3(kWarps * 32), 0, st, a);
    g_trace.launches++;
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "paged attention launch");
}

}  // extern "C"
