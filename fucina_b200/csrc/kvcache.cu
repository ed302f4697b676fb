// Paged key-value cache: rows of f32 keys and values written into f16 or Q8_0 pages, and pages read back as dense rows.
//
// The reference keeps one contiguous f16 or f32 cache per sequence (the operands of src/backend/cuda.zig:2601-2736);
// here the same rows live in pages that a table names, so sequences grow without moving, and Q8_0 halves the bytes the
// attention reads. Q8_0 blocks follow the encoder law of src/backend/quant/q8k.zig:49-69, in its f32 steps, so a cached
// block equals the library's other encoders bit for bit.
//
// Bound: HBM. A written value costs 4 bytes read and 2 (f16) or 1.06 (Q8_0) written, a value read back the cache bytes
// plus 2 or 4. A thread moves eight keys and eight values (a quarter of a Q8_0 block: its scale is agreed over four lanes).
// Measured (B200): 12 000 tokens of eight heads of 128 written as Q8_0 and read back as f16 (225 MB) 48 us = 4.6 TB/s, 71 % of
// a copy's rate; a single token of 32 sequences written and read back 9.1 us, two launches.
#include <cuda_fp16.h>

#include "actquant.cuh"
#include "internal.h"
#include "kvpages.h"
#include "runtime.h"

namespace fq {

int check_kv_pages(const fq_kv_pages* p, KvView* view) {
    if (!p || !p->k || !p->v) return fail(FQ_DECLINED_ARGS, "null key-value pages");
    if (p->fmt != FQ_KV_F16 && p->fmt != FQ_KV_Q8_0) return fail(FQ_DECLINED_ARGS, "cache format %d is not served", p->fmt);
    const bool q8 = p->fmt == FQ_KV_Q8_0;
    if (q8 && (!p->k_scale || !p->v_scale)) return fail(FQ_DECLINED_ARGS, "a Q8_0 cache needs its scale planes");
    if (p->d == 0 || p->d > (size_t)kKvMaxD || p->d % (q8 ? 32 : 16) != 0)
        return fail(FQ_DECLINED_ARGS, "d=%zu: at most %d and a multiple of %d", p->d, kKvMaxD, q8 ? 32 : 16);
    if (p->kv_heads == 0 || p->kv_heads > 512) return fail(FQ_DECLINED_ARGS, "kv_heads=%zu: 1 to 512", p->kv_heads);
    if (p->page_tokens == 0 || p->page_tokens > 4096 || p->page_tokens % 16 != 0)
        return fail(FQ_DECLINED_ARGS, "page_tokens=%zu: a multiple of 16, at most 4096", p->page_tokens);
    if (p->n_pages == 0 || p->n_pages > (size_t)INT32_MAX) return fail(FQ_DECLINED_ARGS, "n_pages out of range");
    const size_t elems = p->kv_heads * p->page_tokens * p->d, scales = elems / 32, most = (size_t)1 << 31;
    if (p->page_stride && (p->page_stride < elems || p->page_stride > most || p->page_stride % (q8 ? 16 : 8) != 0))
        return fail(FQ_DECLINED_ARGS, "page_stride=%zu: shorter than a page, or it breaks the 16-byte alignment", p->page_stride);
    if (q8 && p->scale_stride && (p->scale_stride < scales || p->scale_stride > most || p->scale_stride % 8 != 0))
        return fail(FQ_DECLINED_ARGS, "scale_stride=%zu: shorter than a page's scales, or it breaks the 16-byte alignment", p->scale_stride);
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return fail(FQ_DECLINED_ARGS, "pages must be 16-byte aligned");
    if (q8 && (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 15)) return fail(FQ_DECLINED_ARGS, "scale planes must be 16-byte aligned");
    *view = KvView{(uint8_t*)p->k, (uint8_t*)p->v, (__half*)p->k_scale, (__half*)p->v_scale, (int)p->n_pages, (int)p->page_tokens,
                   (int)p->kv_heads, (int)p->d, p->page_stride ? p->page_stride : elems, p->scale_stride ? p->scale_stride : scales};
    return FQ_OK;
}

namespace {

struct KvRowsArgs {
    KvView c;
    const float* k_in;  // append
    const float* v_in;
    size_t row_stride;
    void* k_out;  // read
    void* v_out;
    const int* seq;
    const int* pos;
    const int* table;
    int n_seqs, max_pages;
    unsigned total;                      // rows * pieces
    FastDiv pieces, head, page_tokens;   // eight-value pieces of a row (kv_heads * d / 8) and of a head (d / 8)
    int* status;
};

// Where piece `col` (eight values) of the row lies: an element offset into k and v, and the block's offset into the scales.
__device__ __forceinline__ void piece_offsets(const KvRowsArgs& A, const KvSlot& at, unsigned col, size_t& elem, size_t& scale) {
    const unsigned head = A.head.div(col), dim = (col - head * A.head.d) * 8;
    const unsigned row = head * A.c.page_tokens + at.slot;
    elem = (size_t)at.page * A.c.page_stride + (size_t)row * A.c.d + dim;
    scale = (size_t)at.page * A.c.scale_stride + row * (A.c.d >> 5) + (dim >> 5);
}

// A thread writes one piece of the keys and the same piece of the values: their loads do not wait for the page table, and
// the address arithmetic is done once for both. (A batch of 11 000 tokens of eight heads of 128, written and read back:
// one piece of one side a thread and plain divisions took 70 us.)
template <bool Q8>
__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ KvRowsArgs A) {
    pdl_wait_then_release();
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    bool live = i < A.total;
    const unsigned row = live ? A.pieces.div(i) : 0, col = live ? i - row * A.pieces.d : 0;
    float k[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = v[j] = 0.0f;
    KvSlot at{-1, 0};
    if (live) {
        const int seq = A.seq[row], pos = A.pos[row];
        load8(A.k_in + (size_t)row * A.row_stride + (size_t)col * 8, k);
        load8(A.v_in + (size_t)row * A.row_stride + (size_t)col * 8, v);
        live = seq >= 0;
        if (live) {
            at = kv_slot(A.table, A.n_seqs, A.max_pages, A.page_tokens, A.c.n_pages, seq, pos);
            if (at.page < 0) {
                *(volatile int*)A.status = FQ_ERR_PAGE;
                live = false;
            }
        }
    }
    size_t elem = 0, sc = 0;
    if (live) piece_offsets(A, at, col, elem, sc);
    if (Q8) {
        // four neighbouring lanes hold a block (a row is whole blocks and the first lane of a warp starts one); every
        // lane takes part in the shuffles, lanes with nothing to write only skip their stores
        int q[8];
        uint2 packed;
        uint16_t dh = q8_0_quarter(k, q);
        packed.x = pack4(q), packed.y = pack4(q + 4);
        if (live) {
            *reinterpret_cast<uint2*>(A.c.k + elem) = packed;
            if ((threadIdx.x & 3) == 0) reinterpret_cast<uint16_t*>(A.c.k_scale)[sc] = dh;
        }
        dh = q8_0_quarter(v, q);
        packed.x = pack4(q), packed.y = pack4(q + 4);
        if (live) {
            *reinterpret_cast<uint2*>(A.c.v + elem) = packed;
            if ((threadIdx.x & 3) == 0) reinterpret_cast<uint16_t*>(A.c.v_scale)[sc] = dh;
        }
    } else if (live) {
        __half2 h[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(k[2 * j], k[2 * j + 1]), h[4 + j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(A.c.k + elem * 2) = *reinterpret_cast<const uint4*>(h);
        *reinterpret_cast<uint4*>(A.c.v + elem * 2) = *reinterpret_cast<const uint4*>(h + 4);
    }
}

// one piece of a side as the output wants it
template <bool Q8, bool HALF_OUT>
__device__ __forceinline__ void write_piece(const uint4& raw, float s, void* out, size_t o) {
    if (!Q8 && HALF_OUT) {
        *reinterpret_cast<uint4*>((__half*)out + o) = raw;
        return;
    }
    float f[8];
    if (Q8) {
        const int8_t* q = reinterpret_cast<const int8_t*>(&raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)q[j] * s;  // 19 bits: exact in f32
    } else {
        const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 x = __half22float2(h[j]);
            f[2 * j] = x.x, f[2 * j + 1] = x.y;
        }
    }
    if (HALF_OUT) {
        __half2 h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
        *reinterpret_cast<uint4*>((__half*)out + o) = *reinterpret_cast<const uint4*>(h);
    } else {
        float* dst = (float*)out + o;
        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
}

template <bool Q8, bool HALF_OUT>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvRowsArgs A) {
    pdl_wait_then_release();
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= A.total) return;
    const unsigned row = A.pieces.div(i), col = i - row * A.pieces.d;
    const int seq = A.seq[row];
    if (seq < 0) return;
    const KvSlot at = kv_slot(A.table, A.n_seqs, A.max_pages, A.page_tokens, A.c.n_pages, seq, A.pos[row]);
    if (at.page < 0) {
        *(volatile int*)A.status = FQ_ERR_PAGE;
        return;
    }
    size_t elem, sc;
    piece_offsets(A, at, col, elem, sc);
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    float ks = 0.0f, vs = 0.0f;
    if (Q8) {
        if (A.k_out) {
            const uint2 x = *reinterpret_cast<const uint2*>(A.c.k + elem);
            k.x = x.x, k.y = x.y, ks = __half2float(A.c.k_scale[sc]);
        }
        if (A.v_out) {
            const uint2 x = *reinterpret_cast<const uint2*>(A.c.v + elem);
            v.x = x.x, v.y = x.y, vs = __half2float(A.c.v_scale[sc]);
        }
    } else {
        if (A.k_out) k = *reinterpret_cast<const uint4*>(A.c.k + elem * 2);
        if (A.v_out) v = *reinterpret_cast<const uint4*>(A.c.v + elem * 2);
    }
    const size_t o = (size_t)i * 8;
    if (A.k_out) write_piece<Q8, HALF_OUT>(k, ks, A.k_out, o);
    if (A.v_out) write_piece<Q8, HALF_OUT>(v, vs, A.v_out, o);
}

int check_rows(const KvView& c, const int32_t* seq, const int32_t* pos, size_t n_tokens, const int32_t* table, size_t n_seqs, size_t max_pages) {
    if (!seq || !pos || !table) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (n_seqs == 0 || n_seqs > (size_t)INT32_MAX || max_pages == 0 || max_pages > (size_t)INT32_MAX / c.page_tokens)
        return fail(FQ_DECLINED_ARGS, "page table of %zu x %zu entries", n_seqs, max_pages);
    if (n_tokens > ((size_t)1 << 33) / ((size_t)c.kv_heads * c.d)) return fail(FQ_DECLINED_ARGS, "more than 2^33 values in one call");
    return FQ_OK;
}

// (total is below 2^30: check_rows)
KvRowsArgs rows_args(const KvView& c, const int32_t* seq, const int32_t* pos, size_t n_tokens, const int32_t* table, size_t n_seqs,
                     size_t max_pages, int* status) {
    KvRowsArgs a{};
    const unsigned pieces = (unsigned)(c.kv_heads * c.d / 8);
    a.c = c, a.seq = seq, a.pos = pos, a.table = table, a.n_seqs = (int)n_seqs, a.max_pages = (int)max_pages;
    a.total = (unsigned)n_tokens * pieces;
    a.pieces = FastDiv(pieces), a.head = FastDiv((unsigned)c.d / 8), a.page_tokens = FastDiv((unsigned)c.page_tokens);
    a.status = status;
    return a;
}

}  // namespace
}  // namespace fq

using namespace fq;

extern "C" {

int fq_kv_append_dev(const fq_kv_pages* pages, const float* k_dev, const float* v_dev, size_t row_stride, const int32_t* token_seq_dev,
                     const int32_t* token_pos_dev, size_t n_tokens, const int32_t* page_table_dev, size_t n_seqs, size_t max_pages, void* stream) {
    KvView c;
    if (int rc = check_kv_pages(pages, &c)) return rc;
    if (n_tokens == 0) return FQ_OK;  // nothing is read: empty buffers may be null
    if (!k_dev || !v_dev) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (int rc = check_rows(c, token_seq_dev, token_pos_dev, n_tokens, page_table_dev, n_seqs, max_pages)) return rc;
    const size_t width = (size_t)c.kv_heads * c.d;
    if (row_stride == 0) row_stride = width;
    if (row_stride < width || row_stride % 4 != 0 || row_stride > ((size_t)1 << 32)) return fail(FQ_DECLINED_ARGS, "row_stride=%zu: at least kv_heads * d and a multiple of 4", row_stride);
    if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) return fail(FQ_DECLINED_ARGS, "k and v must be 16-byte aligned");
    if (!gpu_enabled()) return fail(FQ_DECLINED_GATE, "disabled by FUCINA_GPU=0");
    Ctx* ctx = context();
    if (!ctx) return FQ_DECLINED_NO_GPU;
    std::lock_guard<std::recursive_mutex> g(g_dispatch_lock);
    g_trace.calls++;
    KvRowsArgs a = rows_args(c, token_seq_dev, token_pos_dev, n_tokens, page_table_dev, n_seqs, max_pages, ctx->status_dev);
    a.k_in = k_dev, a.v_in = v_dev, a.row_stride = row_stride;
    const dim3 grid((a.total + 255) / 256);
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    const cudaError_t e = pages->fmt == FQ_KV_Q8_0 ? launch_pdl(kv_append_kernel<true>, grid, dim3(256), 0, st, a)
                                                   : launch_pdl(kv_append_kernel<false>, grid, dim3(256), 0, st, a);
    g_trace.launches++;
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "cache append launch");
}

int fq_kv_read_dev(const fq_kv_pages* pages, void* k_out_dev, void* v_out_dev, int out_is_f16, const int32_t* token_seq_dev,
                   const int32_t* token_pos_dev, size_t n_tokens, const int32_t* page_table_dev, size_t n_seqs, size_t max_pages, void* stream) {
    KvView c;
    if (int rc = check_kv_pages(pages, &c)) return rc;
    if (n_tokens == 0) return FQ_OK;
    if (!k_out_dev && !v_out_dev) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (int rc = check_rows(c, token_seq_dev, token_pos_dev, n_tokens, page_table_dev, n_seqs, max_pages)) return rc;
    if (((uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & 15) return fail(FQ_DECLINED_ARGS, "outputs must be 16-byte aligned");
    if (!gpu_enabled()) return fail(FQ_DECLINED_GATE, "disabled by FUCINA_GPU=0");
    Ctx* ctx = context();
    if (!ctx) return FQ_DECLINED_NO_GPU;
    std::lock_guard<std::recursive_mutex> g(g_dispatch_lock);
    g_trace.calls++;
    KvRowsArgs a = rows_args(c, token_seq_dev, token_pos_dev, n_tokens, page_table_dev, n_seqs, max_pages, ctx->status_dev);
    a.k_out = k_out_dev, a.v_out = v_out_dev;
    const dim3 grid((a.total + 255) / 256);
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    const bool q8 = pages->fmt == FQ_KV_Q8_0;
    const cudaError_t e = q8 ? (out_is_f16 ? launch_pdl(kv_read_kernel<true, true>, grid, dim3(256), 0, st, a)
                                           : launch_pdl(kv_read_kernel<true, false>, grid, dim3(256), 0, st, a))
                             : (out_is_f16 ? launch_pdl(kv_read_kernel<false, true>, grid, dim3(256), 0, st, a)
                                           : launch_pdl(kv_read_kernel<false, false>, grid, dim3(256), 0, st, a));
    g_trace.launches++;
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "cache read launch");
}

}  // extern "C"
