// Attention of one new token per sequence over a paged key-value cache.
//
//   out[s][h] = sum_j softmax_j(scale * q[s][h] . k[j]) v[j],   j in [max(0, len - window), len)
//
// with the running maximum m and sum l of the softmax: keys with scores x change (m, l, o) into
// (m', l e^(m - m') + sum e^(x - m'), o e^(m - m') + sum e^(x - m') v), m' = max(m, x), so K and V are read once. Partial
// results over disjoint keys join the same way.
//
// Bound: HBM, the cache bytes of the keys in range; everything below serves to keep those copies in flight.
//
// Split. Work is counted in units of 16 keys of one kv head (a unit never straddles pages); a row is one (sequence, kv
// head). All units of all rows, in order, are cut into equal shares, one per ring: uneven lengths load the GPU evenly and
// one long sequence uses all of it. A ring is a few shared-memory stages of one unit each, filled by cp.async and walked by
// 1 to 4 warps, each with up to eight of the query heads that share the kv head. A row that lies inside one ring's share
// is finished there; pieces of rows that cross shares are joined inside the CTA in shared memory, and pieces that cross
// CTAs go to the workspace and are joined, in order, by a second kernel. When every row is short, one CTA takes one row
// and no second kernel runs. The lengths are read on the device: nothing on the host depends on them.
//
// Arithmetic. mma.sync m16n8k16 on f16 operands with f32 sums, at f32 accuracy: the operand with 16 rows holds eight heads
// twice, rows 0-7 the leading f16 part of each f32 value and rows 8-15 the remainder (22 bits together), so query and
// weights are not rounded and the split costs no extra instruction; the cache's f16 or int8 values are exact in f16. Query rows are
// scaled by a power of two and weights by 2^15 (their maximum is 1) so that remainders stay clear of f16's smallest steps.
// Q8_0 scales multiply the f32 sums of a 32-value block of a score, and the f32 weights before they are split.
#include <cuda_fp16.h>

#include "internal.h"
#include "kvpages.h"
#include "runtime.h"

namespace fq {

namespace {

constexpr float kNegBig = -3.4e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kUnit = 16;      // keys per unit
constexpr int kRowsPerWarp = 8;
constexpr int kMaxWarps = 8;   // per CTA: up to 255 registers a thread
constexpr int kMaxStages = 8;
constexpr int kSmemMost = 226 * 1024;
constexpr size_t kMaxLen = (size_t)1 << 28;

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
    int passes;        // a kv head with more than 32 query heads is walked in this many rows of `span` heads
    int span;          // query heads of one row
    int warps_per_ring, heads_per_warp, rings, stages;
    int stage_bytes;
    int row_mode;      // one CTA per row; else shares of at least min_units
    int min_units;
    unsigned long long page_magic;  // unit / units per page = unit * page_magic >> 32
    int* meta;         // [grid][2]: the row whose first piece CTA c holds in part 1 (-1: none), the last CTA with a piece of it (in part 0)
    float* parts;      // [grid][2][warps_per_ring * 8][d + 2]: o, then max and sum
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest `newer` groups have landed
__device__ __forceinline__ void cp_async_wait(int newer) {
    switch (newer) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    }
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x, y as f16 leading parts and remainders
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&r);
}
// Two of a word's four int8 values as f16: byte b + 128 becomes the low mantissa bits of 1024 + (b + 128); subtracting 1152
// is exact. sel 0x4140 takes bytes 0 and 1, 0x4342 bytes 2 and 3, 0x4240 the even and 0x4341 the odd ones.
template <int SEL>
__device__ __forceinline__ uint32_t widen(uint32_t biased) {
    const uint32_t u = __byte_perm(biased, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The keys sequence s sees; a length the call does not allow is cut and reported.
__device__ __forceinline__ void key_range(const PagedArgs& A, int s, int& first, int& end) {
    end = A.len[s];
    if (end < 0 || end > A.max_len) {
        *(volatile int*)A.status = FQ_ERR_PAGE;
        end = end < 0 ? 0 : A.max_len;
    }
    first = (A.window > 0 && end > A.window) ? end - A.window : 0;
}
// Units of a row of sequence s: at least one, so that an empty sequence has somebody to write its zeros.
__device__ __forceinline__ int units_of(int first, int end) { return max(1, (end + kUnit - 1) / kUnit - first / kUnit); }

// Where a ring stands: unit `u` of row `r` of sequence `s`.
struct Cursor {
    int s, r, u, units, first, end;
    __device__ __forceinline__ void load(const PagedArgs& A) {
        key_range(A, s, first, end);
        units = units_of(first, end);
    }
    __device__ __forceinline__ void next(const PagedArgs& A, int rows_per_seq) {
        if (++u < units) return;
        u = 0;
        if (++r < rows_per_seq) return;
        r = 0;
        if (++s < A.n_seqs) load(A);
    }
};

// Partial results of a row inside the CTA: two per ring, one of a row that began in an earlier share and one of a row
// that began here and ends in a later one.
struct Piece {
    int row;   // -1: none
    int last;  // the CTA that holds the row's last unit; -1: the unit is in this piece
};

// A sum over both halves of the 16-row operand. Where the leading part met an infinity the remainder's product is
// meaningless (0 or a negative number times infinity).
__device__ __forceinline__ float whole(float lead, float rest) { return fabsf(lead) == INFINITY ? lead : lead + rest; }

template <bool Q8, int DM>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) attn_paged_kernel(const PagedArgs A) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Piece sh_piece[kMaxWarps][2];
    pdl_wait_then_release();
    constexpr int KS = DM / 16;  // 16-value steps of a row
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int ring = warp / A.warps_per_ring, part = warp - ring * A.warps_per_ring;
    const int d = A.c.d, steps = d >> 4;
    const int nc = Q8 ? d >> 4 : d >> 3;   // 16-byte chunks of a key's row
    const int pitch = (nc + 1) * 16;       // an odd number of chunks: the rows of an ldmatrix fall on distinct banks
    const int rows_per_seq = A.c.kv_heads * A.passes;
    const int prow = A.warps_per_ring * kRowsPerWarp;  // head rows of a piece
    const int piece_floats = prow * (d + 2);
    // shared memory: the rings' stages, then one piece per ring; a ring's other piece goes where its stages were
    uint8_t* ring_base = smem + (size_t)ring * A.stages * A.stage_bytes;
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring_base);
    float* pieces_a = reinterpret_cast<float*>(smem + (size_t)A.rings * A.stages * A.stage_bytes);
    auto piece_ptr = [&](int rg, int which) {
        return which == 0 ? pieces_a + (size_t)rg * piece_floats : reinterpret_cast<float*>(smem + (size_t)rg * A.stages * A.stage_bytes);
    };

    // ---- this ring's share
    Cursor cur;
    int count, share = 1;
    long long from = 0;
    if (A.row_mode) {
        cur.s = blockIdx.x / rows_per_seq, cur.r = blockIdx.x - cur.s * rows_per_seq;
        cur.load(A);
        cur.u = (int)((long long)cur.units * ring / A.rings);
        count = (int)((long long)cur.units * (ring + 1) / A.rings) - cur.u;
    } else {
        int mine = 0;
        for (int s = lane; s < A.n_seqs; s += 32) {
            int first, end;
            key_range(A, s, first, end);
            mine += units_of(first, end);
        }
        const int total = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine) * rows_per_seq;
        const int workers = gridDim.x * A.rings;
        share = max(A.min_units, (int)(((long long)total + workers - 1) / workers));
        from = (long long)(blockIdx.x * A.rings + ring) * share;
        count = (int)max(0ll, min((long long)share, total - from));
        cur.s = cur.r = cur.u = 0, cur.units = 1, cur.first = cur.end = 0;
        if (count > 0) {
            // the sequence that holds unit `from`
            int before = 0;
            for (int s0 = 0; s0 < A.n_seqs; s0 += 32) {
                int first = 0, end = 0, n = 0;
                if (s0 + lane < A.n_seqs) key_range(A, s0 + lane, first, end), n = units_of(first, end) * rows_per_seq;
                int sum = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += up;
                }
                const unsigned over = __ballot_sync(0xffffffffu, (long long)before + sum > from);
                if (over) {
                    const int l = __ffs(over) - 1;
                    const int local = (int)(from - before) - __shfl_sync(0xffffffffu, sum - n, l);
                    cur.s = s0 + l;
                    cur.first = __shfl_sync(0xffffffffu, first, l), cur.end = __shfl_sync(0xffffffffu, end, l);
                    cur.units = units_of(cur.first, cur.end);
                    cur.r = local / cur.units, cur.u = local - cur.r * cur.units;
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
    }
    if (part == 0 && lane < 2) sh_piece[ring][lane] = {-1, -1};

    // ---- copies: the ring's warps share the chunks of a unit
    Cursor ahead = cur;
    int to_issue = count;
    int page = -1, page_unit = 0;
    unsigned bad = 0;  // stages whose unit names no page
    auto look_up = [&]() {
        const int ua = ahead.first / kUnit + ahead.u;
        const int slot = (int)(((unsigned long long)(unsigned)ua * A.page_magic) >> 32);
        page_unit = ua - slot * (A.c.page_tokens / kUnit);
        page = ahead.end > 0 ? A.table[(size_t)ahead.s * A.max_pages + slot] : 0;
    };
    const unsigned row_magic = (65536u + nc - 1) / nc;  // chunk / nc = chunk * row_magic >> 16 for chunks < 512
    auto issue = [&](int stage) {
        if (to_issue > 0) {
            const bool ok = page >= 0 && page < A.c.n_pages;
            bad = ok ? bad & ~(1u << stage) : bad | (1u << stage);
            if (!ok) {
                *(volatile int*)A.status = FQ_ERR_PAGE;
            } else if (ahead.end > 0) {
                const size_t tok = (size_t)(ahead.r / A.passes) * A.c.page_tokens + (size_t)page_unit * kUnit;
                const size_t off = ((size_t)page * A.c.page_stride + tok * d) * (Q8 ? 1 : 2);
                const uint32_t dst = ring_addr + stage * A.stage_bytes;
                for (int i = part; i < nc; i += A.warps_per_ring) {  // nc / 2 instructions for the keys, as many for the values
                    const bool side = i >= nc / 2;
                    const int c = lane + 32 * (side ? i - nc / 2 : i), row = (int)((c * row_magic) >> 16);
                    cp_async16(dst + (side ? kUnit * pitch : 0) + (c + row) * 16, (side ? A.c.v : A.c.k) + off + (size_t)c * 16);
                }
                if (Q8 && part == 0 && lane < 2 * (d >> 4)) {  // 16 keys x d / 32 scales = d bytes a side
                    const bool side = lane >= d >> 4;
                    const int c = side ? lane - (d >> 4) : lane;
                    const size_t so = (size_t)page * A.c.scale_stride + tok * (d >> 5);
                    cp_async16(dst + 2 * kUnit * pitch + lane * 16, reinterpret_cast<const uint8_t*>((side ? A.c.v_scale : A.c.k_scale) + so) + c * 16);
                }
            }
            ahead.next(A, rows_per_seq);
            if (--to_issue > 0) look_up();
        }
        cp_async_commit();
    };
    auto ring_sync = [&]() {
        if (A.warps_per_ring == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(ring + 1), "r"(A.warps_per_ring * 32) : "memory");
    };
    if (count > 0) look_up();
    for (int s = 0; s < A.stages - 1; ++s) issue(s);

    // ---- the share, piece by piece
    uint32_t qa[KS][4];
    float o[DM / 8][4], l_run = 0.0f, m_run = -INFINITY, row_scale = 1.0f;
    float v_bound = 0.0f, v_factor = 1.0f;  // Q8_0: values are summed in multiples of the power of two v_bound = 1 / v_factor
    bool started = false;
    int begin_u = 0, stage = 0;
    const int mi = lane >> 3, mr = lane & 7;
    const uint32_t k_lane = (uint32_t)(((mi >> 1) * 8 + mr) * pitch + (mi & 1) * 16);
    const uint32_t v_lane = (uint32_t)(((mi & 1) * 8 + mr) * pitch + (mi >> 1) * 16);

    for (int done = 0; done < count; ++done) {
        if (!started) {
            started = true;
            begin_u = cur.u;
            // query fragments: row g = head g of this warp, times a power of two that puts the row's largest value near 2^14
            const int kvh = cur.r / A.passes, pass = cur.r - kvh * A.passes;
            const int in_row = part * A.heads_per_warp + g, in_group = pass * A.span + in_row;
            const bool live = g < A.heads_per_warp && in_row < A.span && in_group < A.group;
            const float* qrow = A.q + (size_t)cur.s * A.q_stride + (size_t)(kvh * A.group + (live ? in_group : 0)) * d;
            float x[KS][4];
            float big = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[kk][i] = 0.0f;
                if (live && kk < steps) {
                    // f16: columns 2t, 2t + 1, 2t + 8, 2t + 9 of the step; Q8_0: 4t .. 4t + 3, the bytes a lane gets from ldmatrix
                    if (Q8) {
                        const float4 a = *reinterpret_cast<const float4*>(qrow + 16 * kk + 4 * t);
                        x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = a.z, x[kk][3] = a.w;
                    } else {
                        const float2 a = *reinterpret_cast<const float2*>(qrow + 16 * kk + 2 * t), b = *reinterpret_cast<const float2*>(qrow + 16 * kk + 8 + 2 * t);
                        x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = b.x, x[kk][3] = b.y;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(x[kk][i]));
            }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // exponent e of big: rows are multiplied by 2^(14 - e), scores by scale * 2^(e - 14); both factors in two steps so
            // that neither overflows
            const int e = big > 0.0f && big < INFINITY ? (int)((__float_as_uint(big) >> 23) & 255) - 126 : 0;
            const float up = __int_as_float((127 + max(-120, min(120, 14 - e))) << 23);
            const float rest = __int_as_float((127 + (14 - e) - max(-120, min(120, 14 - e))) << 23);
            row_scale = A.scale / up / rest;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                split2(x[kk][0] * up * rest, x[kk][1] * up * rest, qa[kk][0], qa[kk][1]);
                split2(x[kk][2] * up * rest, x[kk][3] * up * rest, qa[kk][2], qa[kk][3]);
            }
            m_run = -INFINITY, l_run = 0.0f, v_bound = 0.0f, v_factor = 1.0f;
#pragma unroll
            for (int n = 0; n < DM / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        }
        cp_async_wait(A.stages - 2);
        ring_sync();  // every warp's copies of this unit have landed, and every warp is done with the stage filled next
        const bool usable = !((bad >> stage) & 1);
        issue(stage == 0 ? A.stages - 1 : stage - 1);

        const int j0 = (cur.first / kUnit + cur.u) * kUnit;
        const int lo = max(cur.first - j0, 0), hi = min(cur.end - j0, kUnit);
        if (usable && hi > lo) {
            const uint32_t ks = ring_addr + stage * A.stage_bytes, vs = ks + kUnit * pitch;
            if (hi - lo < kUnit) {
                // values outside the range may be anything: their rows (Q8_0: their scales) become zeros. The ring's warps write
                // the same zeros.
                uint8_t* rows = ring_base + stage * A.stage_bytes + (Q8 ? 2 * kUnit * pitch + d : kUnit * pitch);
                const int bytes = Q8 ? (d >> 5) * 2 : d * 2, step = Q8 ? (d >> 5) * 2 : pitch;
                for (int r = 0; r < kUnit; ++r)
                    if (r < lo || r >= hi)
                        for (int i = lane * 2; i < bytes; i += 64) *reinterpret_cast<uint16_t*>(rows + r * step + i) = 0;
                __syncwarp();
            }
            // scores of keys 2t, 2t + 1, 2t + 8, 2t + 9 for head g
            float sc[4];
            if (Q8) {
                sc[0] = sc[1] = sc[2] = sc[3] = 0.0f;
                const __half* ksc = reinterpret_cast<const __half*>(ring_base + stage * A.stage_bytes + 2 * kUnit * pitch);
                const int nb = d >> 5;
#pragma unroll
                for (int b = 0; b < KS / 2; ++b) {
                    if (b < nb) {
                        uint32_t r[4];
                        ldsm_x4(ks + k_lane + b * 32, r);  // keys 0-7: values 0-15, 16-31 of the block; keys 8-15: the same
                        float c0[4] = {0, 0, 0, 0}, c1[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
                        mma16816(c0, qa[2 * b], widen<0x4140>(r[0]), widen<0x4342>(r[0]));
                        mma16816(c1, qa[2 * b], widen<0x4140>(r[2]), widen<0x4342>(r[2]));
                        mma16816(c0, qa[2 * b + 1], widen<0x4140>(r[1]), widen<0x4342>(r[1]));
                        mma16816(c1, qa[2 * b + 1], widen<0x4140>(r[3]), widen<0x4342>(r[3]));
                        sc[0] = fmaf(__half2float(ksc[(2 * t) * nb + b]), c0[0] + c0[2], sc[0]);
                        sc[1] = fmaf(__half2float(ksc[(2 * t + 1) * nb + b]), c0[1] + c0[3], sc[1]);
                        sc[2] = fmaf(__half2float(ksc[(2 * t + 8) * nb + b]), c1[0] + c1[2], sc[2]);
                        sc[3] = fmaf(__half2float(ksc[(2 * t + 9) * nb + b]), c1[1] + c1[3], sc[3]);
                    }
                }
            } else {
                float c[2][2][4];
#pragma unroll
                for (int i = 0; i < 16; ++i) (&c[0][0][0])[i] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    if (kk < steps) {
                        uint32_t r[4];
                        ldsm_x4(ks + k_lane + kk * 32, r);  // keys 0-7: values 0-7, 8-15 of the step; keys 8-15: the same
                        mma16816(c[kk & 1][0], qa[kk], r[0], r[1]);
                        mma16816(c[kk & 1][1], qa[kk], r[2], r[3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = i >> 1, x = i & 1;
                    sc[i] = whole(c[0][n][x] + c[1][n][x], c[0][n][x + 2] + c[1][n][x + 2]);
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + (i >> 1) * 8;
                sc[i] = key >= lo && key < hi ? sc[i] * row_scale : -INFINITY;
                top = fmaxf(top, sc[i]);
            }
            // the maximum moves rarely after the first units: the sums are touched only then
            if (__any_sync(0xffffffffu, top > m_run)) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m_run, top);
                const float r = m_run == -INFINITY ? 0.0f : ex2((m_run - m_new) * kLog2e);
                m_run = m_new;
                l_run *= r;
#pragma unroll
                for (int n = 0; n < DM / 8; ++n) o[n][0] *= r, o[n][1] *= r, o[n][2] *= r, o[n][3] *= r;
            }
            float p[4];  // weights times 2^15
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = sc[i] == -INFINITY ? 0.0f : ex2(fmaf(sc[i] - m_run, kLog2e, 15.0f));
                l_run += p[i];
            }
            if (Q8) {
                const int nb = d >> 5;
                const __half* vsc = reinterpret_cast<const __half*>(ring_base + stage * A.stage_bytes + 2 * kUnit * pitch + d);
                // the largest value scale so far, rounded up to a power of two, is taken out of the weights (2^15 times it may
                // pass f16's range) and kept beside the sums
                float most = 0.0f;
                for (int b = 0; b < nb; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = fmaxf(most, __half2float(vsc[(2 * t + (i & 1) + (i >> 1) * 8) * nb + b]));
                if (__any_sync(0xffffffffu, most > v_bound)) {
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    const unsigned bits = (__float_as_uint(fminf(most, 65536.0f)) + 0x7fffffu) & 0xff800000u;
                    const float bound = fmaxf(v_bound, __uint_as_float(bits)), r = v_bound / bound;
                    v_bound = bound;
                    v_factor = 1.0f / bound;
#pragma unroll
                    for (int n = 0; n < DM / 8; ++n) o[n][0] *= r, o[n][1] *= r, o[n][2] *= r, o[n][3] *= r;
                }
#pragma unroll
                for (int b = 0; b < KS / 2; ++b) {
                    if (b < nb) {
                        uint32_t r[4], a[4];
                        ldsm_x4_t(vs + v_lane + b * 32, r);  // values 0-15 of the block: keys 0-7, 8-15; values 16-31: the same
                        const float w0 = p[0] * (__half2float(vsc[(2 * t) * nb + b]) * v_factor), w1 = p[1] * (__half2float(vsc[(2 * t + 1) * nb + b]) * v_factor);
                        const float w2 = p[2] * (__half2float(vsc[(2 * t + 8) * nb + b]) * v_factor), w3 = p[3] * (__half2float(vsc[(2 * t + 9) * nb + b]) * v_factor);
                        split2(w0, w1, a[0], a[1]);
                        split2(w2, w3, a[2], a[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
                        // a lane's word: values 2g, 2g + 1 of key 2t, then of key 2t + 1
                        mma16816(o[4 * b], a, widen<0x4240>(r[0]), widen<0x4240>(r[1]));
                        mma16816(o[4 * b + 1], a, widen<0x4341>(r[0]), widen<0x4341>(r[1]));
                        mma16816(o[4 * b + 2], a, widen<0x4240>(r[2]), widen<0x4240>(r[3]));
                        mma16816(o[4 * b + 3], a, widen<0x4341>(r[2]), widen<0x4341>(r[3]));
                    }
                }
            } else {
                uint32_t a[4];
                split2(p[0], p[1], a[0], a[1]);
                split2(p[2], p[3], a[2], a[3]);
#pragma unroll
                for (int n = 0; n < KS; ++n) {
                    if (n < steps) {
                        uint32_t r[4];
                        ldsm_x4_t(vs + v_lane + n * 32, r);  // values 0-7 of the step: keys 0-7, 8-15; values 8-15: the same
                        mma16816(o[2 * n], a, r[0], r[1]);
                        mma16816(o[2 * n + 1], a, r[2], r[3]);
                    }
                }
            }
        }
        stage = stage + 1 == A.stages ? 0 : stage + 1;

        const bool ended = cur.u + 1 == cur.units;
        if (ended || done + 1 == count) {
            const float l = [&] {
                float x = l_run + __shfl_xor_sync(0xffffffffu, l_run, 1);
                return x + __shfl_xor_sync(0xffffffffu, x, 2);
            }();
            const int row_id = cur.s * rows_per_seq + cur.r;
            const float unit_v = Q8 ? v_bound : 1.0f;
            const int in_row = part * A.heads_per_warp + g;
            if (begin_u == 0 && ended) {
                const int kvh = cur.r / A.passes, in_group = (cur.r - kvh * A.passes) * A.span + in_row;
                if (g < A.heads_per_warp && in_row < A.span && in_group < A.group) {
                    const size_t at = (size_t)cur.s * A.heads + (size_t)kvh * A.group + in_group;
                    const float inv = l > 0.0f || l != l ? unit_v / l : 0.0f;
                    float* dst = A.out + at * d;
#pragma unroll
                    for (int n = 0; n < KS; ++n) {
                        if (n < steps) {
                            if (Q8) {
                                *reinterpret_cast<float4*>(dst + 16 * n + 4 * t) =
                                    make_float4(whole(o[2 * n][0], o[2 * n][2]) * inv, whole(o[2 * n + 1][0], o[2 * n + 1][2]) * inv,
                                                whole(o[2 * n][1], o[2 * n][3]) * inv, whole(o[2 * n + 1][1], o[2 * n + 1][3]) * inv);
                            } else {
                                *reinterpret_cast<float2*>(dst + 16 * n + 2 * t) = make_float2(whole(o[2 * n][0], o[2 * n][2]) * inv, whole(o[2 * n][1], o[2 * n][3]) * inv);
                                *reinterpret_cast<float2*>(dst + 16 * n + 8 + 2 * t) =
                                    make_float2(whole(o[2 * n + 1][0], o[2 * n + 1][2]) * inv, whole(o[2 * n + 1][1], o[2 * n + 1][3]) * inv);
                            }
                        }
                    }
                    if (A.stats && t == 0) A.stats[at * 2] = l > 0.0f ? m_run : kNegBig, A.stats[at * 2 + 1] = l * (1.0f / 32768.0f);
                }
            } else {
                const int which = begin_u != 0 ? 0 : 1;
                if (which == 1) ring_sync();  // the last piece of the share lands on the stages: all warps are done with them
                float* pc = piece_ptr(ring, which) + (size_t)(part * kRowsPerWarp + g) * d;
                float* ml = piece_ptr(ring, which) + (size_t)prow * d + (part * kRowsPerWarp + g) * 2;
#pragma unroll
                for (int n = 0; n < KS; ++n) {
                    if (n < steps) {
                        if (Q8) {
                            float* x = pc + 16 * n + 4 * t;
                            x[0] = whole(o[2 * n][0], o[2 * n][2]) * unit_v, x[1] = whole(o[2 * n + 1][0], o[2 * n + 1][2]) * unit_v;
                            x[2] = whole(o[2 * n][1], o[2 * n][3]) * unit_v, x[3] = whole(o[2 * n + 1][1], o[2 * n + 1][3]) * unit_v;
                        } else {
                            float* x = pc + 16 * n + 2 * t;
                            x[0] = whole(o[2 * n][0], o[2 * n][2]), x[1] = whole(o[2 * n][1], o[2 * n][3]);
                            x[8] = whole(o[2 * n + 1][0], o[2 * n + 1][2]), x[9] = whole(o[2 * n + 1][1], o[2 * n + 1][3]);
                        }
                    }
                }
                if (t == 0) ml[0] = m_run, ml[1] = l;
                const long long last_unit = from + done + (cur.units - 1 - cur.u);
                if (part == 0 && lane == 0) sh_piece[ring][which] = {row_id, ended ? -1 : (int)(last_unit / share / A.rings)};
            }
            started = false;
        }
        cur.next(A, rows_per_seq);
    }

    // ---- join the pieces inside the CTA, in order; what still lacks its beginning or its end goes to the workspace
    __syncthreads();
    const int entries = 2 * A.rings;
    auto entry = [&](int e) { return sh_piece[e >> 1][e & 1]; };
    int tail_row = -1, tail_last = 0;
    for (int e0 = 0; e0 < entries;) {
        const Piece p0 = entry(e0);
        if (p0.row < 0) {
            ++e0;
            continue;
        }
        int e1 = e0 + 1;
        bool ended = p0.last < 0;
        while (e1 < entries && (entry(e1).row < 0 || entry(e1).row == p0.row)) {
            if (entry(e1).row == p0.row) ended = entry(e1).last < 0;
            ++e1;
        }
        const bool begun = (e0 & 1) != 0;
        const int s = p0.row / rows_per_seq, r = p0.row - s * rows_per_seq, kvh = r / A.passes;
        if (begun && !ended) tail_row = p0.row, tail_last = p0.last;
        for (int i = threadIdx.x; i < prow * d; i += blockDim.x) {
            const int pr = i / d, dim = i - pr * d;
            float m = -INFINITY, l = 0.0f, a = 0.0f;
            for (int e = e0; e < e1; ++e)
                if (entry(e).row == p0.row) m = fmaxf(m, piece_ptr(e >> 1, e & 1)[(size_t)prow * d + pr * 2]);
            for (int e = e0; e < e1; ++e)
                if (entry(e).row == p0.row) {
                    const float* pc = piece_ptr(e >> 1, e & 1);
                    const float pm = pc[(size_t)prow * d + pr * 2];
                    const float f = pm == -INFINITY ? 0.0f : ex2((pm - m) * kLog2e);
                    l += pc[(size_t)prow * d + pr * 2 + 1] * f;
                    a += pc[(size_t)pr * d + dim] * f;
                }
            if (begun && ended) {
                const int wp = pr >> 3, in_row = wp * A.heads_per_warp + (pr & 7), in_group = (r - kvh * A.passes) * A.span + in_row;
                if ((pr & 7) < A.heads_per_warp && in_row < A.span && in_group < A.group) {
                    const size_t at = (size_t)s * A.heads + (size_t)kvh * A.group + in_group;
                    A.out[at * d + dim] = l > 0.0f || l != l ? a / l : 0.0f;
                    if (A.stats && dim == 0) A.stats[at * 2] = l > 0.0f ? m : kNegBig, A.stats[at * 2 + 1] = l * (1.0f / 32768.0f);
                }
            } else {
                float* dst = A.parts + ((size_t)blockIdx.x * 2 + (begun ? 1 : 0)) * piece_floats;
                dst[(size_t)pr * d + dim] = a;
                if (dim == 0) dst[(size_t)prow * d + pr * 2] = m, dst[(size_t)prow * d + pr * 2 + 1] = l;
            }
        }
        e0 = e1;
    }
    if (!A.row_mode && threadIdx.x == 0) A.meta[blockIdx.x * 2] = tail_row, A.meta[blockIdx.x * 2 + 1] = tail_last;
}

// Rows that cross CTAs: block (c, head row) joins the row whose beginning CTA c holds with the pieces of the CTAs after it.
// The pieces are added in order by four warps (every fourth piece each), the warps' sums in warp order.
__global__ void __launch_bounds__(128) attn_paged_join_kernel(const PagedArgs A) {
    __shared__ __align__(16) float sh_o[4][kKvMaxD];
    __shared__ float sh_m[4], sh_l[4];
    pdl_wait_then_release();
    const int c0 = blockIdx.x, pr = blockIdx.y, d = A.c.d;
    const int row = A.meta[c0 * 2];
    if (row < 0) return;
    const int rows_per_seq = A.c.kv_heads * A.passes;
    const int s = row / rows_per_seq, r = row - s * rows_per_seq, kvh = r / A.passes;
    const int wp = pr >> 3, in_row = wp * A.heads_per_warp + (pr & 7), in_group = (r - kvh * A.passes) * A.span + in_row;
    if ((pr & 7) >= A.heads_per_warp || in_row >= A.span || in_group >= A.group) return;
    const int prow = A.warps_per_ring * kRowsPerWarp, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t piece_floats = (size_t)prow * (d + 2);
    const int n = A.meta[c0 * 2 + 1] - c0 + 1;
    auto piece = [&](int i) { return A.parts + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * piece_floats; };
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 128) m = fmaxf(m, piece(i)[(size_t)prow * d + pr * 2]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    if (lane == 0) sh_m[w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
    float l = 0.0f;
    for (int d0 = 0; d0 < d; d0 += 128) {
        const int dim = d0 + lane * 4;
        float4 a = make_float4(0, 0, 0, 0);
        for (int i = w; i < n; i += 4) {
            const float* pc = piece(i);
            const float pm = pc[(size_t)prow * d + pr * 2];
            const float f = pm == -INFINITY ? 0.0f : ex2((pm - m) * kLog2e);
            if (d0 == 0) l += pc[(size_t)prow * d + pr * 2 + 1] * f;
            if (dim < d) {
                const float4 x = *reinterpret_cast<const float4*>(pc + (size_t)pr * d + dim);
                a.x = fmaf(x.x, f, a.x), a.y = fmaf(x.y, f, a.y), a.z = fmaf(x.z, f, a.z), a.w = fmaf(x.w, f, a.w);
            }
        }
        if (dim < d) *reinterpret_cast<float4*>(&sh_o[w][dim]) = a;
    }
    if (lane == 0) sh_l[w] = l;
    __syncthreads();
    l = ((sh_l[0] + sh_l[1]) + sh_l[2]) + sh_l[3];
    const size_t at = (size_t)s * A.heads + (size_t)kvh * A.group + in_group;
    for (int i = threadIdx.x; i < d; i += 128) {
        const float a = ((sh_o[0][i] + sh_o[1][i]) + sh_o[2][i]) + sh_o[3][i];
        A.out[at * d + i] = l > 0.0f || l != l ? a / l : 0.0f;
    }
    if (A.stats && threadIdx.x == 0) A.stats[at * 2] = l > 0.0f ? m : kNegBig, A.stats[at * 2 + 1] = l * (1.0f / 32768.0f);
}

// How a call is cut, from sizes the host knows.
struct Plan {
    int passes, span, warps_per_ring, heads_per_warp, rings, stages, stage_bytes;
    int row_mode, grid;
    size_t smem, piece_floats, workspace;
};

// At least two units of a row per share: below that the joins cost more than the copies they spread.
constexpr int kMinUnits = 2;

int plan_paged(const KvView& c, bool q8, size_t n_seqs, size_t heads, size_t max_len, int sm_count, Plan* out) {
    Plan p;
    const int group = (int)heads / c.kv_heads, d = c.d;
    p.passes = (group + 31) / 32;
    p.span = (group + p.passes - 1) / p.passes;
    p.warps_per_ring = (p.span + kRowsPerWarp - 1) / kRowsPerWarp;
    p.heads_per_warp = (p.span + p.warps_per_ring - 1) / p.warps_per_ring;
    const int pitch = ((q8 ? d / 16 : d / 8) + 1) * 16, unit_bytes = kUnit * d * (q8 ? 2 : 4);
    p.stage_bytes = 2 * kUnit * pitch + (q8 ? 2 * d : 0);
    const int piece = p.warps_per_ring * kRowsPerWarp * (d + 2) * (int)sizeof(float);
    // the most rings that still leave 96 KB of copies in flight, else the most bytes in flight
    int best = -1;
    p.rings = p.stages = 0;
    for (int rings = kMaxWarps / p.warps_per_ring; rings >= 1; --rings) {
        int stages = (kSmemMost / rings - piece) / p.stage_bytes;
        stages = stages > kMaxStages ? kMaxStages : stages;
        if (stages < 2 || stages * p.stage_bytes < piece) continue;
        const int flying = rings * (stages - 1) * unit_bytes;
        if (flying > best) best = flying, p.rings = rings, p.stages = stages;
        if (flying >= 96 * 1024) break;
    }
    if (best < 0) return fail(FQ_DECLINED_ARGS, "no shared-memory layout for d=%d and %d heads per kv head", d, group);
    p.smem = (size_t)p.rings * ((size_t)p.stages * p.stage_bytes + piece);
    p.piece_floats = piece / sizeof(float);
    const size_t rows = n_seqs * c.kv_heads * p.passes, units = max_len / kUnit + 2;
    if (rows > (size_t)INT32_MAX / units) return fail(FQ_DECLINED_ARGS, "attention problem too large for one launch");
    p.row_mode = units <= (size_t)8 * p.rings;
    const size_t shares = (rows * units + kMinUnits - 1) / kMinUnits, ctas = (shares + p.rings - 1) / p.rings;
    p.grid = p.row_mode ? (int)rows : (int)(ctas < (size_t)sm_count ? ctas : (size_t)sm_count);
    p.workspace = p.row_mode ? 0 : (size_t)p.grid * 16 + (size_t)p.grid * 2 * p.piece_floats * sizeof(float);
    *out = p;
    return FQ_OK;
}

template <bool Q8, int DM>
cudaError_t launch_paged(const PagedArgs& a, const Plan& p, cudaStream_t st) {
    static bool granted = false;  // under the dispatch lock
    if (!granted) {
        const cudaError_t e = cudaFuncSetAttribute(attn_paged_kernel<Q8, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        if (e != cudaSuccess) return e;
        granted = true;
    }
    return launch_pdl(attn_paged_kernel<Q8, DM>, dim3((unsigned)p.grid), dim3((unsigned)(p.rings * p.warps_per_ring * 32)), p.smem, st, a);
}

int check_paged(const fq_kv_pages* pages, size_t n_seqs, size_t heads, KvView* c) {
    if (int rc = check_kv_pages(pages, c)) return rc;
    if (heads == 0 || heads > 4096 || heads % c->kv_heads != 0)
        return fail(FQ_DECLINED_ARGS, "heads=%zu: a multiple of kv_heads=%d, at most 4096", heads, c->kv_heads);
    if (n_seqs == 0 || n_seqs > 65535) return fail(FQ_DECLINED_ARGS, "n_seqs=%zu: 1 to 65535", n_seqs);
    return FQ_OK;
}

}  // namespace
}  // namespace fq

using namespace fq;

extern "C" {

size_t fq_attn_paged_workspace_bytes(const fq_kv_pages* pages, size_t n_seqs, size_t heads, size_t max_len) {
    KvView c;
    Plan p;
    if (check_paged(pages, n_seqs, heads, &c)) return 0;
    if (max_len > kMaxLen) {
        fail(FQ_DECLINED_ARGS, "max_len=%zu: at most 2^28", max_len);
        return 0;
    }
    Ctx* ctx = context();
    if (!ctx || plan_paged(c, pages->fmt == FQ_KV_Q8_0, n_seqs, heads, max_len, ctx->sm_count, &p)) return 0;
    return p.workspace;
}

int fq_attn_paged_dev(const fq_kv_pages* pages, const float* q_dev, size_t q_stride, const int32_t* page_table_dev, const int32_t* kv_len_dev,
                      size_t n_seqs, size_t max_pages, size_t max_len, size_t heads, float scale, size_t window, float* out_dev,
                      float* stats_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    KvView c;
    if (int rc = check_paged(pages, n_seqs, heads, &c)) return rc;
    if (!q_dev || !page_table_dev || !kv_len_dev || !out_dev) return fail(FQ_DECLINED_ARGS, "null pointer");
    if (max_pages == 0 || max_pages > (size_t)INT32_MAX / c.page_tokens) return fail(FQ_DECLINED_ARGS, "max_pages=%zu out of range", max_pages);
    const size_t capacity = max_pages * c.page_tokens;
    if (max_len == 0 || max_len > capacity) max_len = capacity;
    if (max_len > kMaxLen) return fail(FQ_DECLINED_ARGS, "max_len=%zu: at most 2^28", max_len);
    if (q_stride == 0) q_stride = heads * c.d;
    if (q_stride < heads * c.d || q_stride % 4 != 0 || q_stride > ((size_t)1 << 32)) return fail(FQ_DECLINED_ARGS, "q_stride=%zu: at least heads * d and a multiple of 4", q_stride);
    if (((uintptr_t)q_dev | (uintptr_t)out_dev | (uintptr_t)workspace_dev) & 15) return fail(FQ_DECLINED_ARGS, "q, out and the workspace must be 16-byte aligned");
    if (!gpu_enabled()) return fail(FQ_DECLINED_GATE, "disabled by FUCINA_GPU=0");
    Ctx* ctx = context();
    if (!ctx) return FQ_DECLINED_NO_GPU;
    const bool q8 = pages->fmt == FQ_KV_Q8_0;
    Plan p;
    if (int rc = plan_paged(c, q8, n_seqs, heads, max_len, ctx->sm_count, &p)) return rc;
    if (workspace_dev && workspace_bytes < p.workspace) return fail(FQ_DECLINED_ARGS, "the workspace has %zu of %zu bytes", workspace_bytes, p.workspace);
    std::lock_guard<std::recursive_mutex> g(g_dispatch_lock);
    g_trace.calls++;
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    uint8_t* ws = (uint8_t*)workspace_dev;
    void* own = nullptr;
    if (p.workspace && !ws) {
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(st, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) {
            cudaGetLastError();
            return fail(FQ_DECLINED_ARGS, "a captured call needs a workspace of its own (%zu bytes)", p.workspace);
        }
        own = dev_alloc_on(p.workspace, st);
        if (!own) return fail(FQ_DECLINED_BUDGET, "attention workspace allocation failed");
        ws = (uint8_t*)own;
    }
    if (window > max_len) window = 0;  // it covers every length
    PagedArgs a{};
    a.c = c;
    a.q = q_dev, a.q_stride = q_stride, a.table = page_table_dev, a.len = kv_len_dev;
    a.n_seqs = (int)n_seqs, a.max_pages = (int)max_pages, a.max_len = (int)max_len, a.heads = (int)heads, a.group = (int)heads / c.kv_heads;
    a.scale = scale, a.window = (int)window, a.out = out_dev, a.stats = stats_dev, a.status = ctx->status_dev;
    a.passes = p.passes, a.span = p.span, a.warps_per_ring = p.warps_per_ring, a.heads_per_warp = p.heads_per_warp;
    a.rings = p.rings, a.stages = p.stages, a.stage_bytes = p.stage_bytes, a.row_mode = p.row_mode, a.min_units = kMinUnits;
    const unsigned long long per_page = (unsigned long long)(c.page_tokens / kUnit);
    a.page_magic = ((1ull << 32) + per_page - 1) / per_page;  // exact below 2^32 / 256 units
    a.meta = (int*)ws, a.parts = (float*)(ws + (size_t)p.grid * 16);
    cudaError_t e;
    if (q8) e = c.d <= 64 ? launch_paged<true, 64>(a, p, st) : c.d <= 128 ? launch_paged<true, 128>(a, p, st) : launch_paged<true, 256>(a, p, st);
    else e = c.d <= 64 ? launch_paged<false, 64>(a, p, st) : c.d <= 128 ? launch_paged<false, 128>(a, p, st) : launch_paged<false, 256>(a, p, st);
    g_trace.launches++;
    if (e == cudaSuccess && !p.row_mode) {
        e = launch_pdl(attn_paged_join_kernel, dim3((unsigned)p.grid, (unsigned)(p.warps_per_ring * kRowsPerWarp)), dim3(128), 0, st, a);
        g_trace.launches++;
    }
    if (own) dev_free_on(own, st);
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "paged attention launch");
}

}  // extern "C"
