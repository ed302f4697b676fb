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
// Split. Work is counted in units of 32 keys (16 where a row of K is longer than 128 values) of one kv head; a row is one
// (sequence, kv head). All units of all rows, in order, are cut into chunks; a chunk is walked by one ring: two
// shared-memory stages of one unit each, filled by cp.async and read by 1 to 4 warps, each with up to eight of the query
// heads that share the kv head. A row that lies inside one chunk is finished there; pieces of rows that cross chunks go to
// the workspace and a second kernel joins them in order. The chunks are fixed by the lengths, so a result does not depend on
// which ring walked what. Small calls have one chunk per ring. Large f16 ones, which memory bounds, give each ring one chunk
// of three quarters of its fair share and hand out the rest in small ones as rings become free: SMs differ by a fifth in the
// rate at which memory serves them (64 f16 sequences of up to 8000 tokens: with equal shares the first SM was done after 137
// us, the last after 195; 193.6 us for the call against 198.1). A first kernel then adds up the lengths and clears the
// hand-out counter (the lengths alone where there are many sequences). Q8_0 rings are bound by their own instructions and gain nothing (134 us with equal shares, 148 handed
// out). When every row is short, each row has a team of rings, some of a CTA's, all of them, or those of a cluster of CTAs,
// as the number of rows leaves room (one sequence of 517 tokens: 11.1 us by a CTA a row, 10.2 us by clusters of four); their
// pieces are joined in (distributed) shared memory, and that kernel is the only one. The lengths are read on the device:
// nothing on the host depends on them.
//
// Copies. The keys of a stage are refilled as soon as the scores are taken, the values after the second product: nearly
// two units per ring are in flight at any time from two stages' room.
//
// Arithmetic. mma.sync m16n8k16 on f16 operands with f32 sums, at f32 accuracy: keys (then value columns) are the sixteen
// rows of the first operand, and each query head is two neighbouring columns of the second, the leading f16 part of every
// f32 value and the remainder (22 bits together), so query and weights are not rounded; the cache's f16 or int8 values are
// exact in f16 (an int8 key, raised by 128, as a subnormal: its bits are the integer, and the sum begins with -128 times the
// query's). Four heads fill the eight columns of an instruction (one tile of heads; a warp has one or two): with eight heads
// as rows instead, groups of four heads, the usual ones, leave half of every instruction and half of the softmax empty (64
// Q8_0 sequences of up to 8000 tokens: 152 us, 129 us with heads as columns). A lane holds one head of a tile throughout: its scores of keys g and g + 8, and its sums. Weights change from
// sums to operands by movmatrix. Query rows are scaled by a power of two and weights by 2^15 (their maximum is 1) so that
// remainders stay clear of f16's smallest steps. Q8_0: a key's scale multiplies the f32 sum of its 32-value block; a
// value's scale s turns the two parts (a, b) of a weight into those of the product: a' = a s rounded, b' = b s + (a s - a'),
// whose bracket is exact in f16.
//
// Measured (B200, 32 heads over 8 kv heads of 128): 64 sequences of 300 to 8000 tokens 198 us f16 = 5.50 TB/s, 84 % of a copy's
// rate, and 124-131 us Q8_0 = 4.4-4.7 TB/s; one sequence of 131072 tokens, Q8_0, 67-70 us = 4.1-4.2 TB/s; of 8192 tokens, f16, 18.5 us; of
// 517 tokens 9.8 us. The f16 form waits for memory; the Q8_0 form issues 960 warp instructions per unit, half an instruction
// a cycle and scheduler, and waits for its own results; the small calls are launches and a chain of dependent loads.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "kvpages.h"
#include "runtime.h"

namespace fq {

namespace {

constexpr float kNegBig = -3.4e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSub = 16;       // keys that surely lie in one page
constexpr int kTile = 4;       // query heads of a tile
constexpr int kMaxRings = 16;
constexpr int kSmemMost = 226 * 1024;
constexpr size_t kMaxLen = (size_t)1 << 28;

// Keys per unit and warps per CTA for rows of up to `dm` values and `tiles` tiles of heads a warp: what the registers (the
// sums are tiles * dm / 4 of them, the query half as many) and the stages' room allow.
__host__ __device__ constexpr int unit_keys(int dm) { return dm <= 128 ? 32 : 16; }
__host__ __device__ constexpr int max_warps(int dm, int tiles) { return dm * tiles <= 128 ? 12 : 8; }

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
    int warps_per_ring, heads_per_warp, rows_per_warp, rings;  // rows_per_warp: 4 or 8, heads_per_warp of them in use
    int stage_bytes;
    int row_mode;      // every row has a team of rings
    int team, cluster; // its rings in a CTA, and CTAs
    int planned;       // the plan kernel has run: `sums` holds the units before each sequence
    int dynamic;       // and `next` counts handed-out chunks
    int min_units;     // per chunk
    unsigned page_magic;                  // index of 16 keys / 16-key runs of a page = umulhi(index, page_magic); 0: one run a page
    unsigned page_chunks, scale_chunks;   // 16-byte chunks from page to page
    int* next;
    int* sums;         // [n_seqs + 1]
    int2* meta;        // per chunk: the row that begins in it and ends in a later one (-1: none), the chunk of the row's end
    float* parts;      // per chunk [2][warps_per_ring * rows_per_warp][d + 2] (o, then max and sum): a row that began earlier, a row that ends later
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// the oldest of the four groups under way has landed
__device__ __forceinline__ void cp_async_wait_oldest() { asm volatile("cp.async.wait_group 3;" ::: "memory"); }
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
// the same into fresh sums: `first` in the even columns (heads' leading parts), 0 in the odd ones
__device__ __forceinline__ void mma16816_new(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float first = 0.0f) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(first), "f"(0.0f));
}
// an 8 x 8 matrix of f16, a row's two neighbours per lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float b) {
    float2 r;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// The products of a unit join the running sums by f32 additions: the tensor instruction drops the bits of its sum that do not
// fit, and over a chunk of some hundred instructions those losses, all towards zero, add up (64 f16 sequences of up to 8000
// tokens: 1.7e-6 from the 64-bit result with the running sums inside the instruction, 0.5e-6 apart).
__device__ __forceinline__ void add_to(float (&o)[4], const float (&c)[4]) {
    const float2 a = add2(make_float2(o[0], o[1]), make_float2(c[0], c[1])), b = add2(make_float2(o[2], o[3]), make_float2(c[2], c[3]));
    o[0] = a.x, o[1] = a.y, o[2] = b.x, o[3] = b.y;
}
__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
// x, y as f16 leading parts and remainders
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h), r = add2(make_float2(x, y), make_float2(-f.x, -f.y));
    hi = bits_of(h), lo = bits_of(__floats2half2_rn(r.x, r.y));
}
// A sum over both columns of a head. Where the leading part met an infinity the remainder's product is
// meaningless (0 or a negative number times infinity).
__device__ __forceinline__ float whole(float lead, float rest) {
    const float x = lead + rest;
    return x != x ? lead : x;
}
// Two of a word's four int8 values as f16: byte b + 128 becomes the low mantissa bits of 1024 + (b + 128); subtracting 1152
// is exact. sel 0x4140 takes bytes 0 and 1, 0x4342 bytes 2 and 3, 0x4240 the even and 0x4341 the odd ones.
template <int SEL>
__device__ __forceinline__ uint32_t widen(uint32_t biased) {
    return bits_of(__hsub2(half2_of(__byte_perm(biased, 0x64646464u, SEL)), half2_of(0x64806480u)));
}

// The same as multiples of 2^-24: byte b + 128 as the bits of a subnormal f16, which the product takes exactly. The 128
// times the query's sum is what the block's sum begins with, negative: the terms are some four times the true ones' size in
// the root mean square, which costs two bits of 24 in a block's rounding.
template <int SEL>
__device__ __forceinline__ uint32_t widen_low(uint32_t biased) {
    return __byte_perm(biased, 0u, SEL);
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
// Units of a row: at least one, so that an empty sequence has somebody to write its zeros.
template <int UK>
__device__ __forceinline__ int units_of(int first, int end) {
    return max(1, (end + UK - 1) / UK - first / UK);
}

// Where a ring stands: `left` units of row `r` of sequence `s` are to come, from the keys `key` on.
template <int UK>
struct Cursor {
    int s, r, left, key, first, end;
    __device__ __forceinline__ int units() const { return units_of<UK>(first, end); }
    __device__ __forceinline__ void start_row(int u) { left = units() - u, key = (first / UK + u) * UK; }
    // past a unit; true when that entered another row
    __device__ __forceinline__ bool next(const PagedArgs& A, int rows_per_seq) {
        key += UK;
        if (--left > 0) return false;
        if (++r == rows_per_seq) {
            r = 0;
            if (++s < A.n_seqs) key_range(A, s, first, end);
        }
        start_row(0);
        return true;
    }
};

// How `total` units are cut: `big` units for each of the rings, then chunks of `small`.
struct Cut {
    int total, rings, big, small;
    __device__ __forceinline__ Cut(const PagedArgs& A, int total_, int rings_) : total(total_), rings(rings_) {
        const int fair = (total + rings - 1) / rings;
        big = max(A.min_units, A.dynamic ? fair - fair / 4 : fair);
        small = max(A.min_units, fair / 8);
    }
    // the first unit of chunk c, or the end of all
    __device__ __forceinline__ int begin(int c) const {
        const long long u = c <= rings ? (long long)c * big : (long long)rings * big + (long long)(c - rings) * small;
        return (int)(u < total ? u : total);
    }
    __device__ __forceinline__ int chunk_of(int unit) const {
        const long long over = unit - (long long)rings * big;
        return over < 0 ? unit / big : rings + (int)(over / small);
    }
};

// The scales of one key (or value) row: nb = d / 32 halves, in registers as pairs.
template <int NB, bool EXACT>
__device__ __forceinline__ void load_scales(const __half* row, int nb, uint32_t (&w)[(NB + 1) / 2]) {
    if (EXACT && NB == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(row);
    } else if (EXACT && NB == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(row);
        w[0] = x.x, w[1] = x.y;
    } else if (EXACT && NB == 8) {
        const uint4 x = *reinterpret_cast<const uint4*>(row);
        w[0] = x.x, w[1] = x.y, w[2 % ((NB + 1) / 2)] = x.z, w[3 % ((NB + 1) / 2)] = x.w;
    } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int i = 0; i < (NB + 1) / 2; ++i) w[i] = (2 * i < nb ? h[2 * i] : 0u) | (2 * i + 1 < nb ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    }
}

// EXACT: rows have DM values; else up to DM. HT: tiles of four heads a warp
template <bool Q8, int DM, bool EXACT, int HT>
__global__ void __launch_bounds__(max_warps(DM, HT) * 32, 1) attn_paged_kernel(const __grid_constant__ PagedArgs A) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int sh_next[kMaxRings][2];
    pdl_wait_then_release();
    constexpr int UK = unit_keys(DM);               // keys of a unit
    constexpr int KS = DM / 16, NB = DM / 32;       // 16-value steps and 32-value blocks of a row
    const bool dynamic = !Q8 && A.dynamic;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int ring = warp / A.warps_per_ring, part = warp - ring * A.warps_per_ring;
    const int d = EXACT ? DM : A.c.d, steps = d >> 4, nb = d >> 5;
    const int nc = Q8 ? d >> 4 : d >> 3;  // 16-byte chunks of a key's row
    const int pitch = (nc + 1) * 16;      // an odd number of chunks: the rows of an ldmatrix fall on distinct banks
    const int rows_per_seq = A.c.kv_heads * A.passes;
    constexpr int RPW = kTile * HT;
    const int prow = A.warps_per_ring * RPW;  // head rows of a piece
    const int piece_floats = prow * (d + 2);
    // a stage: K rows, V rows, and for Q8_0 their scales [UK][d / 32]
    const int k_scale_at = 2 * UK * pitch, v_scale_at = k_scale_at + UK * 2 * nb;
    uint8_t* ring_base = smem + (size_t)ring * 2 * A.stage_bytes;
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring_base);
    auto ring_sync = [&]() {
        if (A.warps_per_ring == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(ring + 1), "r"(A.warps_per_ring * 32) : "memory");
    };

    // ---- this ring's first chunk
    Cursor<UK> cur;
    int count, chunk = blockIdx.x * A.rings + ring;
    auto units_total = [&]() {
        if (A.row_mode) return 1;
        if (A.planned) return A.sums[A.n_seqs];
        int mine = 0;
        for (int s = lane; s < A.n_seqs; s += 32) {
            int first, end;
            key_range(A, s, first, end);
            mine += units_of<UK>(first, end);
        }
        return (int)__reduce_add_sync(0xffffffffu, (unsigned)mine) * rows_per_seq;
    };
    const Cut split(A, units_total(), gridDim.x * A.rings);
    // unit `from` of all
    auto locate = [&](Cursor<UK>& c, int from) {
        if (A.planned) {
            // the last sequence with sums[s] <= from: 32 places at a time
            int lo = 0, hi = A.n_seqs;  // sums[lo] <= from < sums[hi]
            while (hi - lo > 1) {
                const int step = (hi - lo + 31) / 32, at = min(lo + lane * step, hi);
                const unsigned below = __ballot_sync(0xffffffffu, at < hi && A.sums[at] <= from);
                const int l = 31 - __clz(below);
                hi = min(lo + (l + 1) * step, hi);
                lo += l * step;
            }
            c.s = lo;
            key_range(A, lo, c.first, c.end);
            from -= A.sums[lo];
        } else {
            for (int s0 = 0; s0 < A.n_seqs; s0 += 32) {
                int first = 0, end = 0, n = 0;
                if (s0 + lane < A.n_seqs) key_range(A, s0 + lane, first, end), n = units_of<UK>(first, end) * rows_per_seq;
                int sum = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += up;
                }
                const unsigned over = __ballot_sync(0xffffffffu, sum > from);
                if (over) {
                    const int l = __ffs(over) - 1;
                    from -= __shfl_sync(0xffffffffu, sum - n, l);
                    c.s = s0 + l;
                    c.first = __shfl_sync(0xffffffffu, first, l), c.end = __shfl_sync(0xffffffffu, end, l);
                    break;
                }
                from -= __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        const int units = c.units();
        c.r = from / units;
        c.start_row(from - c.r * units);
    };
    cur = {0, 0, 1, 0, 0, 0};
    // row_mode: this ring's row and place in the team
    const int teams = A.rings / A.team;
    if (A.row_mode) {
        const int in_cta = ring / A.team, row = blockIdx.x / A.cluster * teams + in_cta;
        count = 0;
        if (in_cta < teams && row < A.n_seqs * rows_per_seq) {
            cur.s = row / rows_per_seq, cur.r = row - cur.s * rows_per_seq;
            key_range(A, cur.s, cur.first, cur.end);
            // a row of few units
            const int units = cur.units(), rank = blockIdx.x % A.cluster * A.team + ring - in_cta * A.team, size = A.cluster * A.team;
            const int u = units * rank / size;
            count = units * (rank + 1) / size - u;
            cur.start_row(u);
            if (part == 0 && lane == 0) sh_next[ring][0] = units;  // for the join
        }
    } else {
        const int from = split.begin(chunk);
        count = split.begin(chunk + 1) - from;
        if (count > 0) locate(cur, from);
        else if (part == 0 && lane == 0 && !dynamic) A.meta[chunk] = make_int2(-1, -1);
    }
    // The chunk after this one is asked for long before it is needed, and the answer is posted to the ring's warps a unit
    // later, when it has arrived; two places, so that none of them finds its answer overwritten. Behind the last chunk of all
    // nobody asks: it may be shorter than the three units that keep asking, posting and reading a barrier apart.
    int asked = 0, answer = 0;
    bool more = false, to_post = false;
    auto ask = [&](int end) {
        more = end < split.total;
        if (!more) return;
        if (part == 0 && lane == 0) answer = split.rings + atomicAdd(A.next, 1);
        ++asked;
        to_post = true;
    };
    auto post = [&]() {
        if (!to_post) return;
        if (part == 0 && lane == 0) sh_next[ring][(asked - 1) & 1] = answer;
        to_post = false;
    };
    if (dynamic && count > 0) ask(split.begin(chunk) + count);

    // ---- copies. `ahead` is the unit copied next; its pages are looked up a step before they are needed. A unit is one or two
    // runs of 16 keys, each inside one page: run x starts `run[x]` chunks into k and v (its scales `srun[x]` chunks into theirs).
    constexpr int RUNS = UK / kSub;
    Cursor<UK> ahead = cur;
    int left = count;
    // the chunk that `ahead` has entered and the ring is yet to begin (a chunk is longer than the two units between them)
    Cursor<UK> coming = cur;
    int coming_chunk = -1, coming_count = 0;
    unsigned have = 0;  // runs of the unit to copy that exist
    unsigned gone_new = 0, gone_next = 0, gone_now = 0;  // runs whose page is no page: of the unit to copy, and of the two in the stages
    struct Look {
        unsigned want;  // runs with keys in range
        int pg[RUNS], at[RUNS];
    };
    size_t run[RUNS], srun[RUNS];
    const int runs_per_page = A.c.page_tokens / kSub;
    const int* table = A.table;
    int head_run = 0;
    auto enter_row = [&]() {
        table = A.table + (size_t)ahead.s * A.max_pages;
        head_run = ahead.r / A.passes * runs_per_page;
    };
    auto look_up = [&](Look& k) {
        k.want = 0;
#pragma unroll
        for (int x = 0; x < RUNS; ++x) {
            const int i = ahead.key / kSub + x;
            k.pg[x] = -1, k.at[x] = 0;
            if (i * kSub < ahead.end && (i + 1) * kSub > ahead.first) {
                const int slot = A.page_magic ? (int)__umulhi((unsigned)i, A.page_magic) : i;
                k.want |= 1u << x;
                k.at[x] = head_run + i - slot * runs_per_page;
                k.pg[x] = table[slot];
            }
        }
    };
    // after the look-up's loads have arrived
    auto place = [&](const Look& k) {
        have = gone_new = 0;
#pragma unroll
        for (int x = 0; x < RUNS; ++x) {
            if ((unsigned)k.pg[x] < (unsigned)A.c.n_pages) {
                have |= 1u << x;
                run[x] = (size_t)(unsigned)k.pg[x] * A.page_chunks + (unsigned)(k.at[x] * kSub * nc);
                if (Q8) srun[x] = (size_t)(unsigned)k.pg[x] * A.scale_chunks + (unsigned)(k.at[x] * nc);
            }
        }
        if (have != k.want) {
            *(volatile int*)A.status = FQ_ERR_PAGE;
            gone_new = have ^ k.want;
        }
    };
    const unsigned row_magic = (65536u + nc - 1) / nc;  // chunk / nc = chunk * row_magic >> 16 for chunks < 512
    const uint32_t copy_dst = ring_addr + (EXACT ? (lane + lane / nc) * 16 : 0);
    const uint8_t* const copy_k = A.c.k + lane * 16;
    const uint8_t* const copy_v = A.c.v + lane * 16;
    // the keys (side 0) or values of the unit to copy into the stage at `stage_at`; the ring's warps take every n-th instruction
    auto copy_side = [&](uint32_t stage_at, int side) {
        if (left > 0) {
#pragma unroll
            for (int x = 0; x < RUNS; ++x) {
                if ((have >> x) & 1) {
                    const uint8_t* src = (side ? copy_v : copy_k) + run[x] * 16;
                    const uint32_t dst = copy_dst + stage_at + (side * UK + x * kSub) * pitch;
                    if (EXACT && A.warps_per_ring == 1) {
#pragma unroll
                        for (int i = 0; i < (Q8 ? DM / 32 : DM / 16); ++i) cp_async16(dst + i * (512 + 512 / nc), src + i * 512);
                    } else if (EXACT) {
                        for (int i = part; i < nc / 2; i += A.warps_per_ring) cp_async16(dst + i * (512 + 512 / nc), src + i * 512);
                    } else {
                        for (int i = part; i < nc / 2; i += A.warps_per_ring) {
                            const int c = lane + 32 * i, row = (int)((c * row_magic) >> 16);
                            cp_async16(dst + (c + row) * 16, src + i * 512);
                        }
                    }
                    if (Q8 && part == 0 && lane < nc)  // 16 keys x d / 32 scales = d bytes
                        cp_async16(ring_addr + stage_at + (side ? v_scale_at : k_scale_at) + x * d + lane * 16,
                                   reinterpret_cast<const uint8_t*>(side ? A.c.v_scale : A.c.k_scale) + srun[x] * 16 + lane * 16);
                }
            }
        }
        cp_async_commit();
    };
    Look look;
    auto step_ahead = [&]() {
        gone_now = gone_next, gone_next = gone_new;
        post();
        if (--left > 0) {
            if (ahead.next(A, rows_per_seq)) enter_row();
            look_up(look);
        } else if (left == 0 && more) {
            const int c = sh_next[ring][(asked - 1) & 1];
            const int from = split.begin(c), n = split.begin(c + 1) - from;
            more = false;
            if (n > 0) {
                locate(ahead, from);
                ask(from + n);
                left = n;
                coming = ahead, coming_chunk = c, coming_count = n;
                enter_row();
                look_up(look);
            }
        }
    };
    // the first two units, both looked up before either is waited for (more than two follow, or none)
    {
        Look first{0, {}, {}}, second{0, {}, {}};
        if (count > 0) enter_row(), look_up(first);
        if (count > 1) {
            if (ahead.next(A, rows_per_seq)) enter_row();
            look_up(second);
        }
        if (left > 0) place(first);
        copy_side(0, 0);
        copy_side(0, 1);
        gone_now = gone_new;
        if (--left > 0) place(second);
        copy_side(A.stage_bytes, 0);
        copy_side(A.stage_bytes, 1);
        gone_next = gone_new, gone_new = 0;
        post();  // a chunk of three units reads the answer in its first step, behind that step's barriers
        if (left > 0 && --left > 0) {
            if (ahead.next(A, rows_per_seq)) enter_row();
            look_up(look);
        }
    }

    // ---- the share, piece by piece
    uint32_t qb[HT][KS][2];
    float q_bias[HT][Q8 ? NB : 1];  // Q8_0: -128 times the sum of a block's query values, in the scores' unit of 2^-24
    float o[HT][DM / 16][4], l_run[HT], m_run[HT], m_use[HT], row_scale[HT];
    float v_cap = 0.0f, v_unit = 1.0f;  // Q8_0: value scales up to v_cap so far; sums count in multiples of v_unit (a power of two)
    __half2 v_norm = half2_of(0x3c003c00u);  // 1 / v_unit
    bool started = false, begun_here = false;
    uint32_t stage_at = 0;
    const int mi = lane >> 3, mr = lane & 7;
    // addresses of a lane in an ldmatrix of four 8 x 8 matrices: (keys, keys + 8) then the next chunk, or the other way round
    const uint32_t by_keys = (uint32_t)(((mi & 1) * 8 + mr) * pitch + (mi >> 1) * 16);
    const uint32_t by_chunks = (uint32_t)(((mi >> 1) * 8 + mr) * pitch + (mi & 1) * 16);

    int done = 0;
    while (count > 0) {
        if (!started) {
            started = true;
            begun_here = cur.key == cur.first / UK * UK;
            // query fragments: column g of tile h = head 4 h + g / 2 of this warp, leading parts (g even) or remainders, times a power
            // of two that puts the row's largest value near 2^14. A lane's sums are those of head 4 h + t: what belongs to a head comes
            // from lane 8 t.
            const int kvh = cur.r / A.passes, pass = cur.r - kvh * A.passes;
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                const int head = kTile * h + (g >> 1), in_row = part * A.heads_per_warp + head, in_group = pass * A.span + in_row;
                const bool live = head < A.heads_per_warp && in_row < A.span && in_group < A.group;
                const float* qrow = A.q + (size_t)cur.s * A.q_stride + (size_t)(kvh * A.group + (live ? in_group : 0)) * d;
                float x[KS][4];
                float big = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[kk][i] = 0.0f;
                    if (live && (EXACT || kk < steps)) {
                        // f16: columns 2t, 2t + 1, 2t + 8, 2t + 9 of the step; Q8_0: 4t .. 4t + 3, the bytes a lane gets from ldmatrix
                        if (Q8) {
                            const float4 a = *reinterpret_cast<const float4*>(qrow + 16 * kk + 4 * t);
                            x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = a.z, x[kk][3] = a.w;
                        } else {
                            const float2 a = *reinterpret_cast<const float2*>(qrow + 16 * kk + 2 * t), b = *reinterpret_cast<const float2*>(qrow + 16 * kk + 8 + 2 * t);
                            x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = b.x, x[kk][3] = b.y;
                        }
                    }
                }
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                    for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(x[kk][i]));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // exponent e of big: rows are multiplied by 2^(14 - e), scores by scale * 2^(e - 14), each in two steps so that no
                // factor overflows
                const int e = big > 0.0f && big < INFINITY ? (int)((__float_as_uint(big) >> 23) & 255) - 126 : 0;
                const int e1 = max(-120, min(120, 14 - e));
                const float up = __int_as_float((127 + e1) << 23), rest = __int_as_float((127 + (14 - e) - e1) << 23);
                row_scale[h] = __shfl_sync(0xffffffffu, A.scale / up / rest, 8 * t);
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    uint32_t hi, low;
                    split2(x[kk][0] * up * rest, x[kk][1] * up * rest, hi, low);
                    qb[h][kk][0] = g & 1 ? low : hi;
                    split2(x[kk][2] * up * rest, x[kk][3] * up * rest, hi, low);
                    qb[h][kk][1] = g & 1 ? low : hi;
                }
                if (Q8) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum += x[2 * b][i] + x[2 * b + 1][i];
                        sum = sum * up * rest;
                        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                        q_bias[h][b] = __shfl_sync(0xffffffffu, sum * (-128.0f / 16777216.0f), 8 * t);
                    }
                }
                m_run[h] = -INFINITY, m_use[h] = 0.0f, l_run[h] = 0.0f;
#pragma unroll
                for (int n = 0; n < DM / 16; ++n) o[h][n][0] = o[h][n][1] = o[h][n][2] = o[h][n][3] = 0.0f;
            }
            v_cap = 0.0f, v_unit = 1.0f;
        }
        const int lo = max(cur.first - cur.key, 0), hi = min(cur.end - cur.key, UK);
        const unsigned lost = gone_now;
        const bool partial = hi - lo < UK || lost;  // some keys do not take part
        const uint32_t ks = ring_addr + stage_at, vs = ks + UK * pitch;
        auto takes_part = [&](int key) { return key >= lo && key < hi && !((lost >> (key / kSub)) & 1); };

        // ---- scores: keys 16 n + g (x) and 16 n + g + 8 (y) for head t of each tile
        cp_async_wait_oldest();
        ring_sync();  // the keys' copies of all the ring's warps have landed
        float2 sc[HT][UK / 16];
        if (Q8) {
            const __half* ksc = reinterpret_cast<const __half*>(ring_base + stage_at + k_scale_at);
#pragma unroll
            for (int n = 0; n < UK / 16; ++n) {
                uint32_t w[2][(NB + 1) / 2];
                load_scales<NB, EXACT>(ksc + (n * 16 + g) * nb, nb, w[0]);
                load_scales<NB, EXACT>(ksc + (n * 16 + g + 8) * nb, nb, w[1]);
#pragma unroll
                for (int h = 0; h < HT; ++h) sc[h][n] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (EXACT || b < nb) {
                        uint32_t r[4];
                        ldsm_x4(ks + n * 16 * pitch + by_keys + b * 32, r);  // values 0-15 of the block: keys 0-7, 8-15; values 16-31: the same
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
                        const uint32_t a0[4] = {widen_low<0x4140>(r[0]), widen_low<0x4140>(r[1]), widen_low<0x4342>(r[0]), widen_low<0x4342>(r[1])};
                        const uint32_t a1[4] = {widen_low<0x4140>(r[2]), widen_low<0x4140>(r[3]), widen_low<0x4342>(r[2]), widen_low<0x4342>(r[3])};
                        const float f0 = (b & 1) ? __high2float(half2_of(w[0][b / 2])) : __low2float(half2_of(w[0][b / 2]));
                        const float f1 = (b & 1) ? __high2float(half2_of(w[1][b / 2])) : __low2float(half2_of(w[1][b / 2]));
#pragma unroll
                        for (int h = 0; h < HT; ++h) {
                            float c[4];
                            mma16816_new(c, a0, qb[h][2 * b][0], qb[h][2 * b][1], q_bias[h][b]);
                            mma16816(c, a1, qb[h][2 * b + 1][0], qb[h][2 * b + 1][1]);
                            sc[h][n].x = fmaf(f0, c[0] + c[1], sc[h][n].x);
                            sc[h][n].y = fmaf(f1, c[2] + c[3], sc[h][n].y);
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int k0 = 0; k0 < KS; k0 += 4) {  // four instructions in a row, then an f32 addition (add_to)
                if (EXACT || k0 < steps) {
                    float c[HT][UK / 16][4];
#pragma unroll
                    for (int kk = k0; kk < k0 + 4; ++kk) {
                        if (EXACT || kk < steps) {
#pragma unroll
                            for (int n = 0; n < UK / 16; ++n) {
                                uint32_t r[4];
                                ldsm_x4(ks + n * 16 * pitch + by_keys + kk * 32, r);  // values 0-7 of the step: keys 0-7, 8-15; values 8-15: the same
#pragma unroll
                                for (int h = 0; h < HT; ++h) {
                                    if (kk == k0) mma16816_new(c[h][n], r, qb[h][kk][0], qb[h][kk][1]);
                                    else mma16816(c[h][n], r, qb[h][kk][0], qb[h][kk][1]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < HT; ++h)
#pragma unroll
                        for (int n = 0; n < UK / 16; ++n) {
                            const float2 part_sum = make_float2(whole(c[h][n][0], c[h][n][1]), whole(c[h][n][2], c[h][n][3]));
                            sc[h][n] = k0 == 0 ? part_sum : add2(sc[h][n], part_sum);
                        }
                }
            }
        }
        ring_sync();  // all the ring's warps are done with the keys
        if (left > 0) place(look);
        copy_side(stage_at, 0);

        // ---- weights
        float top[HT];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < HT; ++h) {
            top[h] = -INFINITY;
#pragma unroll
            for (int n = 0; n < UK / 16; ++n) {
                if (Q8) sc[h][n] = mul2(sc[h][n], 16777216.0f);
                sc[h][n] = mul2(sc[h][n], row_scale[h]);
                if (partial) {
                    if (!takes_part(16 * n + g)) sc[h][n].x = -INFINITY;
                    if (!takes_part(16 * n + g + 8)) sc[h][n].y = -INFINITY;
                }
                top[h] = fmaxf(top[h], fmaxf(sc[h][n].x, sc[h][n].y));
            }
            moved = moved || top[h] > m_run[h];
        }
        // the maximum moves rarely after the first units: the sums are touched only then
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int h = 0; h < HT; ++h) {
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
                const float m_new = fmaxf(m_run[h], top[h]);
                const float r = m_run[h] == -INFINITY ? 0.0f : ex2((m_run[h] - m_new) * kLog2e);
                m_run[h] = m_new;
                m_use[h] = m_new == -INFINITY ? 0.0f : m_new;
                l_run[h] *= r;
#pragma unroll
                for (int n = 0; n < DM / 16; ++n) o[h][n][0] *= r, o[h][n][1] *= r, o[h][n][2] *= r, o[h][n][3] *= r;
            }
        }
        uint32_t ph[HT][UK / 16], pl[HT][UK / 16];  // weights times 2^15 of keys g and g + 8, leading parts and remainders
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int n = 0; n < UK / 16; ++n) {
                const float2 e = fma2(add2(sc[h][n], make_float2(-m_use[h], -m_use[h])), make_float2(kLog2e, kLog2e), make_float2(15.0f, 15.0f));
                const float p0 = ex2(e.x), p1 = ex2(e.y);
                l_run[h] += p0 + p1;
                split2(p0, p1, ph[h][n], pl[h][n]);
            }

        // ---- values
        cp_async_wait_oldest();
        ring_sync();  // the values' copies have landed
        if (partial) {
            // values that do not take part may be anything: their rows (Q8_0: their scales) become zeros. The ring's warps write
            // the same zeros.
            if (Q8) {
                __half* rows = reinterpret_cast<__half*>(ring_base + stage_at + v_scale_at);
                for (int i = lane; i < UK * nb; i += 32)
                    if (!takes_part(i / nb)) rows[i] = __ushort_as_half(0);
            } else {
                for (int i = lane; i < UK * nc; i += 32)
                    if (!takes_part(i / nc)) *reinterpret_cast<uint4*>(ring_base + stage_at + UK * pitch + (i + i / nc) * 16) = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
        }
        if (Q8) {
            const __half* vsc = reinterpret_cast<const __half*>(ring_base + stage_at + v_scale_at);
            uint32_t w[UK / 8][(NB + 1) / 2];
#pragma unroll
            for (int i = 0; i < UK / 8; ++i) load_scales<NB, EXACT>(vsc + (8 * i + g) * nb, nb, w[i]);
            // 2^15 times a scale above 1 may pass f16's range, and products with scales below 2^-9 lose their remainders to f16's
            // smallest steps: then the scales are taken relative to a power of two at or above the largest so far
            __half2 most2 = half2_of(w[0][0]);
#pragma unroll
            for (int i = 0; i < UK / 8; ++i)
#pragma unroll
                for (int b = 0; b < (NB + 1) / 2; ++b) most2 = __hmax2(most2, half2_of(w[i][b]));
            float most = fmaxf(__low2float(most2), __high2float(most2));
            if (__any_sync(0xffffffffu, most > v_cap)) {
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
                float unit = 1.0f;
                v_cap = 1.0f;
                if (most > 1.0f || most <= 1.0f / 512) {
                    const unsigned bits = (__float_as_uint(fmaxf(fminf(most, 65536.0f), 1.0f / 32768)) + 0x7fffffu) & 0xff800000u;
                    unit = v_cap = __uint_as_float(bits);
                }
                const float r = v_unit / unit;
                v_unit = unit;
                v_norm = __float2half2_rn(1.0f / unit);
                // an earlier unit's sums count in the old unit; the cap never falls
#pragma unroll
                for (int h = 0; h < HT; ++h)
#pragma unroll
                    for (int n = 0; n < DM / 16; ++n) o[h][n][0] *= r, o[h][n][1] *= r, o[h][n][2] *= r, o[h][n][3] *= r;
            }
            const bool plain = v_unit == 1.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (EXACT || b < nb) {
                    float c0[HT][4], c1[HT][4];
#pragma unroll
                    for (int n = 0; n < UK / 16; ++n) {
                        __half2 s2 = half2_of(__byte_perm(w[2 * n][b / 2], w[2 * n + 1][b / 2], (b & 1) ? 0x7632 : 0x5410));
                        if (!plain) s2 = __hmul2(s2, v_norm);
                        uint32_t r[4];
                        ldsm_x4_t(vs + n * 16 * pitch + by_keys + b * 32, r);  // values 0-15 of the block: keys 0-7, 8-15; values 16-31: the same
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] ^= 0x80808080u;
                        // a lane's word: values 2g, 2g + 1 of key 2t, then of key 2t + 1: rows g are the even values, rows g + 8 the odd ones
                        const uint32_t a0[4] = {widen<0x4240>(r[0]), widen<0x4341>(r[0]), widen<0x4240>(r[1]), widen<0x4341>(r[1])};
                        const uint32_t a1[4] = {widen<0x4240>(r[2]), widen<0x4341>(r[2]), widen<0x4240>(r[3]), widen<0x4341>(r[3])};
#pragma unroll
                        for (int h = 0; h < HT; ++h) {
                            const __half2 lead = __hmul2(half2_of(ph[h][n]), s2);
                            const __half2 rest = __hfma2(half2_of(pl[h][n]), s2, __hfma2(half2_of(ph[h][n]), s2, __hneg2(lead)));
                            const uint32_t b0 = transposed(__byte_perm(bits_of(lead), bits_of(rest), 0x5410)), b1 = transposed(__byte_perm(bits_of(lead), bits_of(rest), 0x7632));
                            if (n == 0) mma16816_new(c0[h], a0, b0, b1), mma16816_new(c1[h], a1, b0, b1);
                            else mma16816(c0[h], a0, b0, b1), mma16816(c1[h], a1, b0, b1);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < HT; ++h) add_to(o[h][2 * b], c0[h]), add_to(o[h][2 * b + 1], c1[h]);
                }
            }
        } else {
            uint32_t b0[HT][UK / 16], b1[HT][UK / 16];
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int n = 0; n < UK / 16; ++n)
                    b0[h][n] = transposed(__byte_perm(ph[h][n], pl[h][n], 0x5410)), b1[h][n] = transposed(__byte_perm(ph[h][n], pl[h][n], 0x7632));
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if (EXACT || k < steps) {
                    float c[HT][4];
#pragma unroll
                    for (int n = 0; n < UK / 16; ++n) {
                        uint32_t r[4];
                        ldsm_x4_t(vs + n * 16 * pitch + by_chunks + k * 32, r);  // keys 0-7: values 0-7, 8-15 of the step; keys 8-15: the same
#pragma unroll
                        for (int h = 0; h < HT; ++h) {
                            if (n == 0) mma16816_new(c[h], r, b0[h][n], b1[h][n]);
                            else mma16816(c[h], r, b0[h][n], b1[h][n]);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < HT; ++h) add_to(o[h][k], c[h]);
                }
            }
        }
        ring_sync();  // all the ring's warps are done with the values
        copy_side(stage_at, 1);
        step_ahead();
        stage_at = A.stage_bytes - stage_at;

        const bool ended = cur.left == 1, chunk_over = ++done == count;
        if (ended || chunk_over) {
            const int kvh = cur.r / A.passes;
            const bool finished = begun_here && ended;
            const int which = begun_here ? 1 : 0;
            if (A.row_mode && !finished) ring_sync();  // the piece lands on the ring's stages: all its warps are done with them
            float* pc = A.row_mode ? reinterpret_cast<float*>(ring_base) : A.parts + ((size_t)chunk * 2 + which) * piece_floats;
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                float l = l_run[h];
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
                const int head = kTile * h + t, in_row = part * A.heads_per_warp + head, in_group = (cur.r - kvh * A.passes) * A.span + in_row;
                const bool live = head < A.heads_per_warp && in_row < A.span && in_group < A.group;
                const size_t at = (size_t)cur.s * A.heads + (size_t)kvh * A.group + in_group;
                float* dst = finished ? A.out + at * d : pc + (size_t)(part * RPW + head) * d;
                const float f = finished ? (l > 0.0f || l != l ? v_unit / l : 0.0f) : v_unit;
                if (live || !finished) {
#pragma unroll
                    for (int n = 0; n < KS; ++n) {
                        if (EXACT || n < steps) {
                            const float a = whole(o[h][n][0], o[h][n][1]) * f, b = whole(o[h][n][2], o[h][n][3]) * f;
                            if (Q8) *reinterpret_cast<float2*>(dst + 16 * n + 2 * g) = make_float2(a, b);
                            else dst[16 * n + g] = a, dst[16 * n + g + 8] = b;
                        }
                    }
                }
                if (finished) {
                    if (A.stats && live && g == 0) A.stats[at * 2] = l > 0.0f ? m_run[h] : kNegBig, A.stats[at * 2 + 1] = l * (1.0f / 32768.0f);
                } else if (g == 0) {
                    float* ml = pc + (size_t)prow * d + (part * RPW + head) * 2;
                    ml[0] = m_run[h], ml[1] = l;
                }
            }
            if (!finished && which == 1 && !A.row_mode && part == 0 && lane == 0)
                A.meta[chunk] = make_int2(cur.s * rows_per_seq + cur.r, split.chunk_of(split.begin(chunk) + done - 1 + cur.left - 1));
            if (chunk_over && !A.row_mode && (finished || which == 0) && part == 0 && lane == 0) A.meta[chunk] = make_int2(-1, -1);
            started = false;
        }
        if (!chunk_over) {
            cur.next(A, rows_per_seq);
        } else {
            done = 0, count = 0;
            if (coming_chunk >= 0) cur = coming, chunk = coming_chunk, count = coming_count, coming_chunk = -1;
        }
    }
    if (!A.row_mode) return;

    // ---- join the teams' pieces, in order: a warp per (row, head row), a lane per piece for the weights (two where a team has
    // more than 32 rings), then four values a lane, eight pieces at a time
    namespace cg = cooperative_groups;
    if (A.cluster > 1) cg::this_cluster().sync();
    else __syncthreads();
    const int size = A.cluster * A.team, warps = blockDim.x >> 5, cta = blockIdx.x % A.cluster;
    const int ring_floats = 2 * A.stage_bytes / (int)sizeof(float);
    for (int item = cta + A.cluster * warp; item < teams * prow && size > 1; item += A.cluster * warps) {
        const int in_cta = item / prow, pr = item - in_cta * prow, row = blockIdx.x / A.cluster * teams + in_cta;
        if (row >= A.n_seqs * rows_per_seq) continue;
        const int s = row / rows_per_seq, r = row - s * rows_per_seq, kvh = r / A.passes;
        const int in_row = pr / RPW * A.heads_per_warp + pr % RPW, in_group = (r - kvh * A.passes) * A.span + in_row;
        if (pr % RPW >= A.heads_per_warp || in_row >= A.span || in_group >= A.group) continue;
        const int units = sh_next[in_cta * A.team][0];
        if (units == 1) continue;  // finished by its ring
        // ring k of the team's part in CTA c
        float* const here = reinterpret_cast<float*>(smem) + in_cta * A.team * ring_floats;
        auto pieces_of = [&](int c) { return A.cluster > 1 ? (const float*)cg::this_cluster().map_shared_rank(here, c) : (const float*)here; };
        float m[2], l[2], f[2], m_all = -INFINITY, l_all = 0.0f;
        unsigned present[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int k = lane + 32 * x;
            const bool in = k < size && units * (k + 1) / size > units * k / size;
            m[x] = -INFINITY, l[x] = 0.0f;
            if (in) {
                const int c = A.cluster > 1 ? k / A.team : 0;
                const float2 ml = *reinterpret_cast<const float2*>(pieces_of(c) + (k - c * A.team) * ring_floats + prow * d + pr * 2);
                m[x] = ml.x, l[x] = ml.y;
            }
            present[x] = __ballot_sync(0xffffffffu, in);
            m_all = fmaxf(m_all, m[x]);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, x));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            f[x] = m[x] == -INFINITY ? 0.0f : ex2((m[x] - m_all) * kLog2e);
            l_all += l[x] * f[x];
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) l_all += __shfl_xor_sync(0xffffffffu, l_all, x);
        const size_t at = (size_t)s * A.heads + (size_t)kvh * A.group + in_group;
        const float inv = l_all > 0.0f || l_all != l_all ? 1.0f / l_all : 0.0f;
        for (int i0 = 0; i0 < d; i0 += 128) {
            const int i = i0 + lane * 4;
            float4 a = make_float4(0, 0, 0, 0);
            for (int c = 0; c < A.cluster; ++c) {
                const float* p = pieces_of(c) + pr * d + i;
                for (int k0 = 0; k0 < A.team; k0 += 4) {
                    float4 v[4];
                    float fk[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int kk = c * A.team + k0 + k;
                        const bool there = k0 + k < A.team && (((kk < 32 ? present[0] : present[1]) >> (kk & 31)) & 1);
                        fk[k] = __shfl_sync(0xffffffffu, kk < 32 ? f[0] : f[1], kk & 31);
                        if (!there) fk[k] = 0.0f;
                        v[k] = there && i < d ? *reinterpret_cast<const float4*>(p + (k0 + k) * ring_floats) : make_float4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        a.x = fmaf(v[k].x, fk[k], a.x), a.y = fmaf(v[k].y, fk[k], a.y), a.z = fmaf(v[k].z, fk[k], a.z), a.w = fmaf(v[k].w, fk[k], a.w);
                }
            }
            if (i < d) *reinterpret_cast<float4*>(A.out + at * d + i) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        }
        if (lane == 0 && A.stats) A.stats[at * 2] = l_all > 0.0f ? m_all : kNegBig, A.stats[at * 2 + 1] = l_all * (1.0f / 32768.0f);
    }
    if (A.cluster > 1) cg::this_cluster().sync();  // no CTA leaves while another reads its pieces
}

// The units before each sequence, and a fresh hand-out counter: one CTA, 1024 sequences at a time.
template <int UK>
__global__ void __launch_bounds__(1024) attn_paged_plan_kernel(const PagedArgs A) {
    __shared__ int sh_warp[32];
    pdl_wait_then_release();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows_per_seq = A.c.kv_heads * A.passes;
    if (threadIdx.x == 0) *A.next = 0;
    int before = 0;
    for (int s0 = 0; s0 < A.n_seqs; s0 += 1024) {
        const int s = s0 + threadIdx.x;
        int first, end, n = 0;
        if (s < A.n_seqs) key_range(A, s, first, end), n = units_of<UK>(first, end) * rows_per_seq;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31) sh_warp[warp] = sum;
        __syncthreads();
        int base = lane < warp ? sh_warp[lane] : 0, all = sh_warp[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o), all += __shfl_xor_sync(0xffffffffu, all, o);
        if (s < A.n_seqs) A.sums[s] = before + base + sum - n;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) A.sums[A.n_seqs] = before;
}

// Rows that cross chunks. Work items are (chunk, head row); a block of eight warps first finds, 256 at a time, which of its
// items begin a row that ends in a later chunk. A row of up to 16 pieces is joined by one warp, a longer one by all eight,
// every eighth piece a warp, and the warps' results in warp order. Loads are what bounds this: a lane loads the maximum and
// the sum of one piece, 32 pieces at once, and then four values of eight pieces before any of them is used.
constexpr int kJoinWarps = 8, kJoinAlone = 16;
struct Joined {
    float m, l;
    float4 a[kKvMaxD / 128];
    __device__ __forceinline__ void scale(float f) {
        l *= f;
#pragma unroll
        for (int x = 0; x < kKvMaxD / 128; ++x) a[x].x *= f, a[x].y *= f, a[x].z *= f, a[x].w *= f;
    }
};
__global__ void __launch_bounds__(kJoinWarps * 32) attn_paged_join_kernel(const PagedArgs A, int rings) {
    __shared__ __align__(16) float sh_o[kJoinWarps][kKvMaxD];
    __shared__ float sh_m[kJoinWarps], sh_l[kJoinWarps];
    __shared__ int4 sh_todo[kJoinWarps * 32];
    __shared__ int sh_count[2];
    pdl_wait_then_release();
    const int d = A.c.d, w = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = kJoinWarps * 32;
    const int prow = A.warps_per_ring * A.rows_per_warp, rows_per_seq = A.c.kv_heads * A.passes;
    const size_t piece_floats = (size_t)prow * (d + 2);
    int chunks = rings;
    if (A.dynamic) {
        const Cut split(A, A.sums[A.n_seqs], rings);
        chunks = split.chunk_of(split.total - 1) + 1;
    }
    // pieces from, from + step, .. of item (chunk, head row, row, last chunk)
    auto join = [&](const int4& it, int from, int step) {
        const int n = it.w - it.x + 1, pr = it.y;
        Joined j{-INFINITY, 0.0f, {}};
        for (int i0 = from; i0 < n; i0 += 32 * step) {
            const int mine = i0 + lane * step, count = min(32, (n - i0 + step - 1) / step);
            auto piece = [&](int i) { return A.parts + ((size_t)(it.x + i) * 2 + (i == 0 ? 1 : 0)) * piece_floats; };
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (mine < n) ml = *reinterpret_cast<const float2*>(piece(mine) + (size_t)prow * d + pr * 2);
            float m = fmaxf(j.m, ml.x);
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            j.scale(j.m == -INFINITY ? 0.0f : ex2((j.m - m) * kLog2e));
            j.m = m;
            const float f = ml.x == -INFINITY ? 0.0f : ex2((ml.x - m) * kLog2e);
            float l = ml.y * f;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            j.l += l;
            for (int k0 = 0; k0 < count; k0 += 8) {
#pragma unroll
                for (int x = 0; x < kKvMaxD / 128; ++x) {
                    const int dim = x * 128 + lane * 4;
                    if (x * 128 >= d) break;
                    float4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        v[k] = k0 + k < count && dim < d ? *reinterpret_cast<const float4*>(piece(i0 + (k0 + k) * step) + (size_t)pr * d + dim) : make_float4(0, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float fk = __shfl_sync(0xffffffffu, f, k0 + k);
                        if (k0 + k < count) j.a[x].x = fmaf(v[k].x, fk, j.a[x].x), j.a[x].y = fmaf(v[k].y, fk, j.a[x].y), j.a[x].z = fmaf(v[k].z, fk, j.a[x].z), j.a[x].w = fmaf(v[k].w, fk, j.a[x].w);
                    }
                }
            }
        }
        return j;
    };
    // where item `it` goes: the head's place in out, or -1
    auto place_of = [&](const int4& it) {
        const int s = it.z / rows_per_seq, r = it.z - s * rows_per_seq, kvh = r / A.passes;
        const int in_row = it.y / A.rows_per_warp * A.heads_per_warp + it.y % A.rows_per_warp, in_group = (r - kvh * A.passes) * A.span + in_row;
        if (it.y % A.rows_per_warp >= A.heads_per_warp || in_row >= A.span || in_group >= A.group) return -1ll;
        return (long long)s * A.heads + (long long)kvh * A.group + in_group;
    };
    const long long items = (long long)chunks * prow;
    for (long long base = blockIdx.x; base < items; base += (long long)gridDim.x * threads) {
        if (threadIdx.x < 2) sh_count[threadIdx.x] = 0;
        __syncthreads();
        const long long item = base + (long long)threadIdx.x * gridDim.x;
        if (item < items) {
            const int c = (int)(item / prow);
            const int2 m = A.meta[c];
            // from the front those for one warp, from the back those for all: any order, the items are independent
            if (m.x >= 0) {
                const int4 it = make_int4(c, (int)(item - (long long)c * prow), m.x, m.y);
                if (m.y - c + 1 <= kJoinAlone) sh_todo[atomicAdd(&sh_count[0], 1)] = it;
                else sh_todo[threads - 1 - atomicAdd(&sh_count[1], 1)] = it;
            }
        }
        __syncthreads();
        const int alone = sh_count[0], together = sh_count[1];
        for (int k = w; k < alone; k += kJoinWarps) {
            const int4 it = sh_todo[k];
            const long long at = place_of(it);
            if (at < 0) continue;
            const Joined j = join(it, 0, 1);
            const float inv = j.l > 0.0f || j.l != j.l ? 1.0f / j.l : 0.0f;
#pragma unroll
            for (int x = 0; x < kKvMaxD / 128; ++x) {
                const int dim = x * 128 + lane * 4;
                if (dim < d) *reinterpret_cast<float4*>(A.out + at * d + dim) = make_float4(j.a[x].x * inv, j.a[x].y * inv, j.a[x].z * inv, j.a[x].w * inv);
            }
            if (A.stats && lane == 0) A.stats[at * 2] = j.l > 0.0f ? j.m : kNegBig, A.stats[at * 2 + 1] = j.l * (1.0f / 32768.0f);
        }
        for (int k = 0; k < together; ++k) {
            const int4 it = sh_todo[threads - 1 - k];
            const long long at = place_of(it);
            if (at < 0) continue;
            const Joined j = join(it, w, kJoinWarps);
#pragma unroll
            for (int x = 0; x < kKvMaxD / 128; ++x)
                if (x * 128 + lane * 4 < d) *reinterpret_cast<float4*>(&sh_o[w][x * 128 + lane * 4]) = j.a[x];
            if (lane == 0) sh_m[w] = j.m, sh_l[w] = j.l;
            __syncthreads();
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int i = 0; i < kJoinWarps; ++i) m = fmaxf(m, sh_m[i]);
            float f[kJoinWarps];
#pragma unroll
            for (int i = 0; i < kJoinWarps; ++i) f[i] = sh_m[i] == -INFINITY ? 0.0f : ex2((sh_m[i] - m) * kLog2e), l += sh_l[i] * f[i];
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            for (int i = threadIdx.x; i < d; i += threads) {
                float a = 0.0f;
#pragma unroll
                for (int x = 0; x < kJoinWarps; ++x) a += sh_o[x][i] * f[x];
                A.out[at * d + i] = a * inv;
            }
            if (A.stats && threadIdx.x == 0) A.stats[at * 2] = l > 0.0f ? m : kNegBig, A.stats[at * 2 + 1] = l * (1.0f / 32768.0f);
            __syncthreads();  // sh_o, sh_m and sh_l are free for the next item
        }
        __syncthreads();
    }
}

// How a call is cut, from sizes the host knows.
struct Plan {
    int dm, exact, tiles, passes, span, warps_per_ring, heads_per_warp, rings, stage_bytes;
    int row_mode, team, cluster, planned, dynamic, grid, chunks;
    size_t smem, sums_at, meta_at, parts_at, workspace;
};

// A chunk has at least two units (a ring's depth of copies; below that the joins cost more than the copies they spread),
// three where chunks are handed out.
constexpr int kMinUnits = 2, kMinUnitsDynamic = 3;

// Up to this many sequences every ring adds up the lengths itself, 32 at a time, in less than the launch of a kernel that
// does it for all; beyond, the plan kernel runs.
constexpr size_t kPlanSeqs = 512;


// Teams walk rows of at most this many units per ring, longer ones are better spread over all rings: where the teams leave
// SMs idle (one sequence of 4000 tokens, eight kv heads, f16: 18.5 us by teams of 24 rings, 5.3 units each, 15.0 us over all
// rings), and where they fill three quarters of the GPU (16 sequences of 2000 tokens, Q8_0: 22.0 us by teams, 27.4 us over all
// rings).
constexpr int kTeamUnits = 4, kTeamUnitsFull = 8;

int plan_paged(const KvView& c, bool q8, size_t n_seqs, size_t heads, size_t max_len, int sm_count, Plan* out) {
    Plan p;
    const int group = (int)heads / c.kv_heads, d = c.d;
    p.exact = d == 64 || d == 128 || d == 256;
    p.dm = d <= 64 && p.exact ? 64 : d <= 128 ? 128 : 256;
    p.passes = (group + 31) / 32;
    p.span = (group + p.passes - 1) / p.passes;
    p.tiles = p.span <= kTile ? 1 : 2;
    const int rows_per_warp = kTile * p.tiles;
    p.warps_per_ring = (p.span + rows_per_warp - 1) / rows_per_warp;
    p.heads_per_warp = (p.span + p.warps_per_ring - 1) / p.warps_per_ring;
    const int keys = unit_keys(p.dm), pitch = ((q8 ? d / 16 : d / 8) + 1) * 16;
    p.stage_bytes = 2 * keys * pitch + (q8 ? 4 * keys * (d / 32) : 0);
    const size_t piece = (size_t)p.warps_per_ring * rows_per_warp * (d + 2) * sizeof(float);
    // as many rings as warps and two stages each allow
    p.rings = max_warps(p.dm, p.tiles) / p.warps_per_ring;
    while (p.rings > 1 && p.rings * 2 * p.stage_bytes > kSmemMost) --p.rings;
    if (p.rings * 2 * p.stage_bytes > kSmemMost) return fail(FQ_DECLINED_ARGS, "no shared-memory layout for d=%d and %d heads per kv head", d, group);
    p.smem = (size_t)p.rings * 2 * p.stage_bytes;
    const size_t rows = n_seqs * c.kv_heads * p.passes, units = max_len / keys + 2;
    if (rows > ((size_t)INT32_MAX - 65536) / units) return fail(FQ_DECLINED_ARGS, "attention problem too large for one launch");
    // Teams: the most rings per row with which all rows run at once; whole CTAs where that leaves half the SMs idle, up to a
    // cluster of four (a team of 64 rings at most is joined by one warp).
    p.team = p.rings, p.cluster = 1;
    while (p.team > 1 && (rows + p.rings / p.team - 1) / (p.rings / p.team) > (size_t)sm_count) --p.team;
    while (p.cluster < 4 && p.team == p.rings && 2 * rows * p.cluster <= (size_t)sm_count && units > (size_t)p.team * p.cluster) p.cluster *= 2;
    // (a piece of a team lies on its ring's stages)
    const bool full = 4 * ((rows + p.rings / p.team - 1) / (p.rings / p.team)) * p.cluster >= 3 * (size_t)sm_count;
    p.row_mode = units <= (size_t)(full ? kTeamUnitsFull : kTeamUnits) * p.team * p.cluster && (p.team * p.cluster == 1 || (size_t)2 * p.stage_bytes >= piece);
    if (!p.row_mode) p.team = p.rings, p.cluster = 1;
    const size_t most = rows * units, rings_all = (size_t)sm_count * p.rings;
    p.dynamic = !p.row_mode && !q8 && most >= 48 * rings_all;
    p.planned = !p.row_mode && (p.dynamic || n_seqs > kPlanSeqs);
    const size_t shares = (most + kMinUnits - 1) / kMinUnits, ctas = (shares + p.rings - 1) / p.rings;
    p.grid = p.row_mode ? (int)((rows + p.rings / p.team - 1) / (p.rings / p.team)) * p.cluster : (int)(ctas < (size_t)sm_count ? ctas : (size_t)sm_count);
    // one chunk per ring; handed out, the rest (a quarter of the fair shares) in chunks of an eighth of one or of three units:
    // (fair / 4) / (fair / 8) rounded down is at most 5 / 1, and 3 where the least size binds
    p.chunks = p.grid * p.rings * (p.dynamic ? 6 : 1);
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.sums_at = 256;
    p.meta_at = p.sums_at + (p.planned ? up((n_seqs + 1) * sizeof(int)) : 0);
    p.parts_at = p.meta_at + up(p.chunks * sizeof(int2));
    p.workspace = p.row_mode ? 0 : p.parts_at + (size_t)p.chunks * 2 * piece;
    *out = p;
    return FQ_OK;
}

template <bool Q8, int DM, bool EXACT, int HT>
cudaError_t launch_paged(const PagedArgs& a, const Plan& p, cudaStream_t st) {
    static bool granted = false;  // under the dispatch lock
    if (!granted) {
        const cudaError_t e = cudaFuncSetAttribute(attn_paged_kernel<Q8, DM, EXACT, HT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        if (e != cudaSuccess) return e;
        granted = true;
    }
    const dim3 grid((unsigned)p.grid), block((unsigned)(p.rings * p.warps_per_ring * 32));
    if (p.cluster == 1) return launch_pdl(attn_paged_kernel<Q8, DM, EXACT, HT>, grid, block, p.smem, st, a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = p.smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    static const bool no_pdl = getenv("FUCINA_B200_NO_PDL") != nullptr;
    cfg.attrs = attr, cfg.numAttrs = no_pdl ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, attn_paged_kernel<Q8, DM, EXACT, HT>, a);
}
template <bool Q8, int HT>
cudaError_t launch_paged(const PagedArgs& a, const Plan& p, cudaStream_t st) {
    if (p.dm == 64) return launch_paged<Q8, 64, true, HT>(a, p, st);
    if (p.dm == 128) return p.exact ? launch_paged<Q8, 128, true, HT>(a, p, st) : launch_paged<Q8, 128, false, HT>(a, p, st);
    return p.exact ? launch_paged<Q8, 256, true, HT>(a, p, st) : launch_paged<Q8, 256, false, HT>(a, p, st);
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
    a.passes = p.passes, a.span = p.span, a.warps_per_ring = p.warps_per_ring, a.heads_per_warp = p.heads_per_warp, a.rows_per_warp = kTile * p.tiles;
    a.rings = p.rings, a.stage_bytes = p.stage_bytes, a.row_mode = p.row_mode, a.team = p.team, a.cluster = p.cluster, a.planned = p.planned, a.dynamic = p.dynamic;
    a.min_units = p.dynamic ? kMinUnitsDynamic : kMinUnits;
    const unsigned long long per_page = (unsigned long long)(c.page_tokens / kSub);
    a.page_magic = per_page == 1 ? 0 : (unsigned)(((1ull << 32) + per_page - 1) / per_page);  // exact below 2^32 / 256 runs of 16 keys
    a.page_chunks = (unsigned)(c.page_stride / (q8 ? 16 : 8)), a.scale_chunks = (unsigned)(c.scale_stride / 8);
    a.next = (int*)ws, a.sums = (int*)(ws + p.sums_at), a.meta = (int2*)(ws + p.meta_at), a.parts = (float*)(ws + p.parts_at);
    cudaError_t e = cudaSuccess;
    if (p.planned) {
        e = launch_pdl(unit_keys(p.dm) == 32 ? attn_paged_plan_kernel<32> : attn_paged_plan_kernel<16>, dim3(1), dim3(1024), 0, st, a);
        g_trace.launches++;
    }
    if (e == cudaSuccess) e = p.tiles == 1 ? (q8 ? launch_paged<true, 1>(a, p, st) : launch_paged<false, 1>(a, p, st)) : q8 ? launch_paged<true, 2>(a, p, st) : launch_paged<false, 2>(a, p, st);
    g_trace.launches++;
    if (e == cudaSuccess && !p.row_mode) {
        const size_t items = (size_t)p.chunks * p.warps_per_ring * a.rows_per_warp, blocks = (size_t)ctx->sm_count * 4;
        e = launch_pdl(attn_paged_join_kernel, dim3((unsigned)(items < blocks ? items : blocks)), dim3(kJoinWarps * 32), 0, st, a, p.grid * p.rings);
        g_trace.launches++;
    }
    if (own) dev_free_on(own, st);
    return e == cudaSuccess ? FQ_OK : cuda_fail(e, "paged attention launch");
}

}  // extern "C"
