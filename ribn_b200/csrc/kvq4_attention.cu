// Attention over the 4-bit paged KV cache (kvq4.cuh): a few query rows per sequence against long key ranges.
//
// A CTA of four warps takes a span of pages of one (sequence, kv head) for a block of up to 8 or 16 columns (column = row of the
// sequence x query head of the group); warp w takes pages w, w + 4, .. and is a pipeline of its own: page records come into its
// ring of shared memory by asynchronous copies, kRing - 1 pages ahead.  With m16n8k16 products, per page of 16 keys:
//   S^T = K Q^T   a masked nibble is a binary16 number by itself, code x 2^-24 (or, one nibble up, 2^-20: those dimensions' queries
//                 are held 2^-4 times), so a word of eight codes costs a shift and four masks and no conversion.  A group of 32
//                 dimensions is summed apart, beginning with -8 x the sum of its queries, and enters the score times its scale.
//                 Queries are scaled by a power of two per column, so that binary16 holds F16 and BF16 ones exactly.
//   O^T = V^T P^T a nibble under the exponent of 64 is 64 + code; one fused multiply-add with the scale and -72 x scale, both exact,
//                 gives the value.  P comes from the S^T layout by transposing 8 x 8 blocks across the warp.
// F32 queries and their probabilities are binary16 hi + lo pairs (two products each).  Softmax in base 2; a column's reference moves
// only when a score passes it by 2^8, and P is held 2^7 times, so that small probabilities stay normal numbers.
// The spans' sums meet in a merge kernel in span order: results do not depend on where pages lie or on other sequences' keys.
#include <math.h>

#include <algorithm>

#include "kvq4.cuh"

namespace ribn {

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHeld = 7.0f;    // P is held 2^7 times ..
constexpr float kSlack = 8.0f;   // .. and may grow to 2^15

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t bits_of(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 half2_of(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t other) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(other));
    return r;
}
// d = a b + c
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 2) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    } else {
        static_assert(WORDS % 4 == 0, "whole 16-byte reads");
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(addr + 4 * i));
        }
    }
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ void store_value(const KvQ4Attention& a, long long at, float x) {
    if (a.type == kQ4F32) static_cast<float*>(a.out)[at] = x;
    else if (a.type == kQ4F16) static_cast<__half*>(a.out)[at] = __float2half_rn(x);
    else asm volatile("{\n\t.reg .b16 t;\n\tcvt.rn.bf16.f32 t, %1;\n\tst.global.b16 [%0], t;\n\t}" ::"l"(static_cast<unsigned short*>(a.out) + at), "f"(x) : "memory");
}

// The rows of a sequence and the pages that a block of its columns sees.  Positions: row i is at base + i.
struct Block {
    int row0, n, base, cols, first_row, last_row;
    int low, high;         // keys that some row of the block sees: low <= key < high
    int page0, pages, per, spans;
};
__device__ __forceinline__ Block block_of(const KvQ4Attention& a, int s, int cb) {
    Block b;
    const int group = a.q_heads / a.kv_heads;
    b.row0 = max(a.cu_rows[s], 0);
    b.n = min(a.cu_rows[s + 1], a.rows) - b.row0;
    const int length = min(max(a.lengths[s], 0), a.pages_per_sequence * kQ4Page);
    b.base = length - b.n;
    b.cols = (long long)b.n * group > a.tile_above ? 0 : max(0, min(a.span_cols, b.n * group - cb * a.span_cols));   // 0: the tile kernel's
    b.first_row = cb * a.span_cols / group;
    b.last_row = (cb * a.span_cols + b.cols - 1) / group;
    b.high = max(0, b.base + b.last_row + 1);
    b.low = a.window > 0 ? max(0, b.base + b.first_row - a.window + 1) : 0;
    b.page0 = b.low / kQ4Page;
    b.pages = b.high > b.low ? (b.high + kQ4Page - 1) / kQ4Page - b.page0 : 0;
    b.per = max(a.span_pages, (b.pages + a.max_spans - 1) / a.max_spans);
    b.spans = max(1, (b.pages + b.per - 1) / b.per);
    return b;
}

constexpr int kRing = 4;   // page records per warp: one read, three on their way

// NT: column tiles of 8.  PAIR: F32 queries.
template <int HD, int NT, bool PAIR>
__global__ void __launch_bounds__(kWarps * 32, HD <= 128 && NT == 1 ? (PAIR ? 3 : 4) : 2) kvq4_span_kernel(const KvQ4Attention a) {
    constexpr int NG = HD / 32, WORDS = NG < 4 ? NG : 4, SUB = NG / WORDS;
    constexpr int RECORD = q4_record(HD), RING = kRing, REC = HD + 2;
    constexpr int BLOCK = kQ4Page * 16 * WORDS;   // bytes of codes of one sub
    extern __shared__ __align__(128) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.q_heads / a.kv_heads;
    // (span, sequence, kv head, column block), the last one fastest
    int id = blockIdx.x;
    const int cb = id % a.col_blocks; id /= a.col_blocks;
    const int kvh = id % a.kv_heads; id /= a.kv_heads;
    const int s = id % a.sequences, span = id / a.sequences;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Block b = block_of(a, s, cb);
    if (b.cols <= 0 || span >= b.spans) return;
    const int begin = b.page0 + span * b.per, end = min(begin + b.per, b.page0 + b.pages);
    const int mine = max(0, (end - begin - warp + kWarps - 1) / kWarps);   // this warp's pages
    const int32_t* table = a.page_tables + s * a.table_stride + begin + warp;
    const uint32_t ring = smem_at(smem) + warp * (RING * RECORD);
    const unsigned char* head = a.cache + (long long)kvh * RECORD;
    const long long page_stride = (long long)a.kv_heads * RECORD;

    // Page i of this warp: its number lies in lane i % 32; one outside of the arena is neither copied nor seen.
    int ids = lane < mine ? table[lane * kWarps] : -1;
    uint32_t good = 0;   // by i % 32
    auto issue = [&](int i) {
        if (i < mine) {
            if (i > 0 && (i & 31) == 0) ids = i + lane < mine ? table[(i + lane) * kWarps] : -1;
            const int page = __shfl_sync(0xffffffffu, ids, i & 31);
            const bool ok = page >= 0 && page < a.pages;
            good = (good & ~(1u << (i & 31))) | ((uint32_t)ok << (i & 31));
            if (ok) {
                const unsigned char* from = head + page * page_stride + lane * 16;
                const uint32_t to = ring + (i % RING) * RECORD + lane * 16;
#pragma unroll
                for (int o = 0; o < RECORD; o += 512) {
                    if (o + 512 <= RECORD || lane * 16 < RECORD - o) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + o), "l"(from + o) : "memory");
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) issue(i);

    // B fragments of Q^T: column 8 nt + g; of group G the dimensions 32 G + 8 t + {0, 4, 2, 6} and, 2^-4 times, {1, 5, 3, 7}
    uint32_t qh[NT][NG][4], ql[PAIR ? NT : 1][PAIR ? NG : 1][4];
    float start[NT][NG][2], factor[NT][2];
    int last[NT][2], lowest[NT][2];   // keys that columns 8 nt + 2 t + {0, 1} see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + g, flat = cb * a.span_cols + col;
        const bool have = col < b.cols;
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int G = 0; G < NG; ++G) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[G][i] = 0.0f;
            if (have) q4_load8(a.q, (b.row0 + flat / group) * a.q_stride + (long long)(kvh * group + flat % group) * HD + 32 * G + 8 * t, a.type, a.vector_q, x[G]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[G][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e brings the largest to [2^13, 2^14)
        const int e = top > 0.0f && top < INFINITY ? max(-126, min(126, 140 - (int)(__float_as_uint(top) >> 23))) : 0;
        const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
        const float f = down * (a.scale * kLog2e * 16777216.0f);
        factor[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
        factor[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int G = 0; G < NG; ++G) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[G][i] *= up; sum += x[G][i]; }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= -8.0f / 16777216.0f;
            start[nt][G][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
            start[nt][G][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = (u & 1) * 2 + (u >> 1);   // 0, 2, 1, 3: the word's pairs are (i, i + 4)
                const float m = (u >> 1) ? 0.0625f : 1.0f;
                const __half2 h = __floats2half2_rn(x[G][i] * m, x[G][i + 4] * m);
                qh[nt][G][u] = bits_of(h);
                if (PAIR) {
                    const float2 back = __half22float2(h);
                    ql[PAIR ? nt : 0][PAIR ? G : 0][u] = bits_of(__floats2half2_rn(x[G][i] * m - back.x, x[G][i + 4] * m - back.y));
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int at = nt * 8 + 2 * t + c;
            last[nt][c] = at < b.cols ? b.base + (cb * a.span_cols + at) / group : -1;
            lowest[nt][c] = a.window > 0 ? last[nt][c] - a.window + 1 : 0;
        }
    }
    // keys that every column sees
    const int all_low = a.window > 0 ? b.base + b.last_row - a.window + 1 : 0, all_high = b.base + b.first_row;

    float o[NT][2 * NG][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < 2 * NG; ++mt) { o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f; }
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
    }

    for (int i = 0; i < mine; ++i) {
        issue(i + RING - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
        __syncwarp();
        if (!((good >> (i & 31)) & 1u)) continue;
        const uint32_t page = ring + (i % RING) * RECORD;
        const int key0 = (begin + warp + kWarps * i) * kQ4Page;
        const bool masked = key0 < all_low || key0 + kQ4Page - 1 > all_high;
        // ---- scores of keys g (values 0, 1) and g + 8 (values 2, 3), columns 8 nt + 2 t + {0, 1}
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
        {
            uint32_t s0[NG / 2], s1[NG / 2];
            if constexpr (NG == 2) {
                s0[0] = lds32(page + 16 * HD + g * 4); s1[0] = lds32(page + 16 * HD + (g + 8) * 4);
            } else {
                lds_words<NG / 2>(page + 16 * HD + g * (2 * NG), s0);
                lds_words<NG / 2>(page + 16 * HD + (g + 8) * (2 * NG), s1);
            }
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                uint32_t w0[WORDS], w1[WORDS];
                lds_words<WORDS>(page + sub * BLOCK + lane * (4 * WORDS), w0);
                lds_words<WORDS>(page + sub * BLOCK + BLOCK / 2 + lane * (4 * WORDS), w1);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const int G = sub * WORDS + w;
                    const uint32_t x0 = w0[w] >> 8, x1 = w1[w] >> 8;
                    const uint32_t even[4] = {w0[w] & 0x000F000Fu, w1[w] & 0x000F000Fu, x0 & 0x000F000Fu, x1 & 0x000F000Fu};
                    const uint32_t odd[4] = {w0[w] & 0x00F000F0u, w1[w] & 0x00F000F0u, x0 & 0x00F000F0u, x1 & 0x00F000F0u};
                    const float2 k0 = __half22float2(half2_of(s0[G >> 1])), k1 = __half22float2(half2_of(s1[G >> 1]));
                    const float f0 = (G & 1) ? k0.y : k0.x, f1 = (G & 1) ? k1.y : k1.x;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float from[4] = {start[nt][G][0], start[nt][G][1], start[nt][G][0], start[nt][G][1]};
                        float acc[4];
                        if (PAIR) {
                            const uint32_t(&lo)[4] = ql[PAIR ? nt : 0][PAIR ? G : 0];
                            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma(acc, even, lo[0], lo[1], zero);
                            mma(acc, odd, lo[2], lo[3], acc);
                            float high[4];
                            mma(high, even, qh[nt][G][0], qh[nt][G][1], from);
                            mma(high, odd, qh[nt][G][2], qh[nt][G][3], high);
#pragma unroll
                            for (int u = 0; u < 4; ++u) acc[u] += high[u];
                        } else {
                            mma(acc, even, qh[nt][G][0], qh[nt][G][1], from);
                            mma(acc, odd, qh[nt][G][2], qh[nt][G][3], acc);
                        }
                        sc[nt][0] = fmaf(acc[0], f0, sc[nt][0]); sc[nt][1] = fmaf(acc[1], f0, sc[nt][1]);
                        sc[nt][2] = fmaf(acc[2], f1, sc[nt][2]); sc[nt][3] = fmaf(acc[3], f1, sc[nt][3]);
                    }
                }
            }
        }
        // ---- softmax
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            sc[nt][0] *= factor[nt][0]; sc[nt][1] *= factor[nt][1]; sc[nt][2] *= factor[nt][0]; sc[nt][3] *= factor[nt][1];
            if (masked) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int key = key0 + g + 8 * (u >> 1);
                    if (key > last[nt][u & 1] || key < lowest[nt][u & 1]) sc[nt][u] = -INFINITY;
                }
            }
            over = over || fmaxf(sc[nt][0], sc[nt][2]) > m[nt][0] + kSlack || fmaxf(sc[nt][1], sc[nt][3]) > m[nt][1] + kSlack;
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(sc[nt][c], sc[nt][2 + c]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    f[c] = 1.0f;
                    if (top > m[nt][c] + kSlack || (m[nt][c] == -INFINITY && top > -INFINITY)) {
                        f[c] = m[nt][c] == -INFINITY ? 0.0f : exp2_approx(m[nt][c] - top);
                        m[nt][c] = top;
                    }
                    l[nt][c] *= f[c];
                }
#pragma unroll
                for (int mt = 0; mt < 2 * NG; ++mt) { o[nt][mt][0] *= f[0]; o[nt][mt][1] *= f[1]; o[nt][mt][2] *= f[0]; o[nt][mt][3] *= f[1]; }
            }
        }
        uint32_t ph[NT][2], pl[PAIR ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0] - kHeld, m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1] - kHeld;
            const float p0 = exp2_approx(sc[nt][0] - m0), p1 = exp2_approx(sc[nt][1] - m1), p2 = exp2_approx(sc[nt][2] - m0), p3 = exp2_approx(sc[nt][3] - m1);
            l[nt][0] += p0 + p2; l[nt][1] += p1 + p3;
            const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
            ph[nt][0] = movmatrix_trans(bits_of(h0)); ph[nt][1] = movmatrix_trans(bits_of(h1));
            if (PAIR) {
                const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                pl[PAIR ? nt : 0][0] = movmatrix_trans(bits_of(__floats2half2_rn(p0 - b0.x, p1 - b0.y)));
                pl[PAIR ? nt : 0][1] = movmatrix_trans(bits_of(__floats2half2_rn(p2 - b1.x, p3 - b1.y)));
            }
        }
        // ---- values: dimensions 32 G + g + {0, 8} and {16, 24}, keys 2 t + {0, 1} and + 8
        {
            uint32_t s0[NG], s1[NG];
            lds_words<NG>(page + 17 * HD + t * (4 * NG), s0);
            lds_words<NG>(page + 17 * HD + (4 + t) * (4 * NG), s1);
            if (masked) {   // what lies where no row looks may be anything
                const int k = key0 + 2 * t;
                const uint32_t keep0 = (k >= b.low && k < b.high ? 0xffffu : 0u) | (k + 1 >= b.low && k + 1 < b.high ? 0xffff0000u : 0u);
                const uint32_t keep1 = (k + 8 >= b.low && k + 8 < b.high ? 0xffffu : 0u) | (k + 9 >= b.low && k + 9 < b.high ? 0xffff0000u : 0u);
#pragma unroll
                for (int G = 0; G < NG; ++G) { s0[G] &= keep0; s1[G] &= keep1; }
            }
            const __half2 minus72 = __float2half2_rn(-72.0f);
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                uint32_t w0[WORDS], w1[WORDS];
                lds_words<WORDS>(page + 8 * HD + sub * BLOCK + lane * (4 * WORDS), w0);
                lds_words<WORDS>(page + 8 * HD + sub * BLOCK + BLOCK / 2 + lane * (4 * WORDS), w1);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const int G = sub * WORDS + w;
                    const __half2 a0 = half2_of(s0[G]), a1 = half2_of(s1[G]), b0 = __hmul2(a0, minus72), b1 = __hmul2(a1, minus72);
                    auto value = [&](uint32_t x, __half2 sa, __half2 sb) { return bits_of(__hfma2(half2_of(and_or(x, 0x00F000F0u, 0x54005400u)), sa, sb)); };
                    const uint32_t lower[4] = {value(w0[w] << 4, a0, b0), value(w0[w], a0, b0), value(w1[w] << 4, a1, b1), value(w1[w], a1, b1)};
                    const uint32_t upper[4] = {value(w0[w] >> 4, a0, b0), value(w0[w] >> 8, a0, b0), value(w1[w] >> 4, a1, b1), value(w1[w] >> 8, a1, b1)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (PAIR) {   // a page's sum by itself: the instruction cuts at the last bit of what it adds to
                            float lo[4] = {0.0f, 0.0f, 0.0f, 0.0f}, up[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma(lo, lower, pl[PAIR ? nt : 0][0], pl[PAIR ? nt : 0][1], lo);
                            mma(up, upper, pl[PAIR ? nt : 0][0], pl[PAIR ? nt : 0][1], up);
                            mma(lo, lower, ph[nt][0], ph[nt][1], lo);
                            mma(up, upper, ph[nt][0], ph[nt][1], up);
#pragma unroll
                            for (int u = 0; u < 4; ++u) { o[nt][2 * G][u] += lo[u]; o[nt][2 * G + 1][u] += up[u]; }
                        } else {
                            mma(o[nt][2 * G], lower, ph[nt][0], ph[nt][1], o[nt][2 * G]);
                            mma(o[nt][2 * G + 1], upper, ph[nt][0], ph[nt][1], o[nt][2 * G + 1]);
                        }
                    }
                }
            }
        }
        __syncwarp();   // every lane has read the slot before the next copies land in it
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // ---- the warps' sums meet in shared memory, in warp order
    constexpr int kWarpFloats = RING * RECORD / 4;
    static_assert(kWarpFloats >= 8 * NT * REC, "a warp's ring holds its columns' sums");
    float* rec = reinterpret_cast<float*>(smem) + warp * kWarpFloats;
    if (mine > 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = nt * 8 + 2 * t + c;
                float sum = l[nt][c];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (col < b.cols) {
#pragma unroll
                    for (int G = 0; G < NG; ++G) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) rec[col * REC + 32 * G + 8 * u + g] = o[nt][2 * G + (u >> 1)][2 * (u & 1) + c];
                    }
                    if (g == 0) { rec[col * REC + HD] = m[nt][c]; rec[col * REC + HD + 1] = sum; }
                }
            }
        }
    }
    __syncthreads();
    const int live = min(kWarps, end - begin);
    const float* recs = reinterpret_cast<const float*>(smem);
    for (int col = warp; col < b.cols; col += kWarps) {
        const int flat = cb * a.span_cols + col, row = b.row0 + flat / group, qh_index = kvh * group + flat % group;
        float top = -INFINITY;
        for (int w = 0; w < live; ++w) top = fmaxf(top, recs[w * kWarpFloats + col * REC + HD]);
        float acc[HD / 32], total = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
        for (int w = 0; w < live; ++w) {
            const float mw = recs[w * kWarpFloats + col * REC + HD], fw = mw == -INFINITY ? 0.0f : exp2_approx(mw - top);
            total = fmaf(recs[w * kWarpFloats + col * REC + HD + 1], fw, total);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(recs[w * kWarpFloats + col * REC + lane + 32 * i], fw, acc[i]);
        }
        if (b.spans == 1) {
            const long long at = row * a.out_stride + (long long)qh_index * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) store_value(a, at + lane + 32 * i, total > 0.0f || total != total ? acc[i] / total : 0.0f);
        } else {
            float* pp = a.partial + (((long long)row * a.q_heads + qh_index) * a.max_spans + span) * REC;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) pp[lane + 32 * i] = acc[i];
            if (lane == 0) { pp[HD] = top; pp[HD + 1] = total; }
        }
    }
}

// out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M): four warps per (row, query head), warp w spans w, w + 4, .., then the warps in order.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) kvq4_merge_kernel(const KvQ4Attention a) {
    constexpr int DPL = HD / 32, REC = HD + 2, GROUP = 4;
    __shared__ float sums[kWarps][HD + 1];
    const int row = (int)blockIdx.x / a.q_heads, qh = (int)blockIdx.x % a.q_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = a.q_heads / a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int s = 0, above = a.sequences;   // the last sequence that begins at or before the row
    while (above - s > 1) {
        const int mid = (s + above) / 2;
        if (a.cu_rows[mid] <= row) s = mid; else above = mid;
    }
    if (row < a.cu_rows[s] || row >= a.cu_rows[s + 1]) return;
    const int flat = (row - a.cu_rows[s]) * group + qh % group;
    if (flat / a.span_cols >= a.col_blocks) return;   // more rows than the call said
    const Block b = block_of(a, s, flat / a.span_cols);
    if (b.cols <= 0 || b.spans <= 1) return;   // written by the tile or the span kernel
    const float* pp = a.partial + ((long long)row * a.q_heads + qh) * a.max_spans * REC;
    float top = -INFINITY;
    for (int i = lane; i < b.spans; i += 32) top = fmaxf(top, __ldcg(pp + (long long)i * REC + HD));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum[DPL], denom = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) sum[i] = 0.0f;
    for (int s0 = warp; s0 < b.spans; s0 += kWarps * GROUP) {
        float v[GROUP][DPL], mx[GROUP], lx[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const int at = s0 + kWarps * u;
            const float* rec = pp + (long long)at * REC;
#pragma unroll
            for (int i = 0; i < DPL; ++i) v[u][i] = at < b.spans ? __ldcg(rec + lane + 32 * i) : 0.0f;
            mx[u] = at < b.spans ? __ldcg(rec + HD) : -INFINITY;
            lx[u] = at < b.spans ? __ldcg(rec + HD + 1) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const float w = mx[u] == -INFINITY ? 0.0f : exp2_approx(mx[u] - top);
            denom = fmaf(lx[u], w, denom);
#pragma unroll
            for (int i = 0; i < DPL; ++i) sum[i] = fmaf(v[u][i], w, sum[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < DPL; ++i) sums[warp][lane + 32 * i] = sum[i];
    if (lane == 0) sums[warp][HD] = denom;
    __syncthreads();
    const float total = ((sums[0][HD] + sums[1][HD]) + sums[2][HD]) + sums[3][HD];
    for (int d = threadIdx.x; d < HD; d += kWarps * 32) {
        const float value = ((sums[0][d] + sums[1][d]) + sums[2][d]) + sums[3][d];
        store_value(a, row * a.out_stride + (long long)qh * HD + d, total > 0.0f || total != total ? value / total : 0.0f);
    }
}

bool aligned16(const void* p, long long stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; }

// How a launch is split: columns per CTA and spans.
void plan_spans(KvQ4Attention& a) {
    const int group = a.q_heads / a.kv_heads;
    a.tile_above = a.head_dim == 256 ? 0x7fffffff : 32;
    const int cols = (int)std::min<long long>((long long)std::min(a.max_rows, a.rows) * group, a.tile_above);
    // 16 columns share a page's conversion; with heads of 256 their sums do not fit in the registers (1,080 bytes of spills)
    a.span_cols = cols <= 8 || a.head_dim == 256 ? 8 : 16;
    a.col_blocks = (cols + a.span_cols - 1) / a.span_cols;
    const int keys = a.window > 0 ? (int)std::min<long long>(a.max_keys, (long long)a.window + a.max_rows + kQ4Page) : a.max_keys;
    const int pages = std::max(1, (keys + kQ4Page - 1) / kQ4Page);
    const long long items = (long long)a.sequences * a.kv_heads * a.col_blocks;
    const long long resident = (long long)kvq4_sm_count() * (a.head_dim <= 128 && a.span_cols == 8 ? (a.type == kQ4F32 ? 3 : 4) : 2);
    // F32: a sum of at most 16 pages per warp, as each addition of the matrix instruction cuts at the sum's last bit
    const int most = a.type == kQ4F32 ? 64 : 1 << 20;
    // the fewest page-times of the busiest CTA, with a span's set-up and fold counted as eight pages of a warp
    float best = 0.0f;
    a.span_pages = std::min(pages, most);
    for (int spans = (pages + most - 1) / most; spans <= std::min(512, (pages + 3) / 4); spans += std::max(1, spans / 8)) {
        const int per = (pages + spans - 1) / spans;
        const long long waves = (items * spans + resident - 1) / resident;
        const float cost = (float)waves * ((float)((per + 3) / 4) + 8.0f) + (spans > 1 ? 6.0f + 0.5f * (float)(spans / 16) : 0.0f);
        if (best == 0.0f || cost < best) { best = cost; a.span_pages = per; }
    }
    a.max_spans = (pages + a.span_pages - 1) / a.span_pages;
}

template <typename Kernel>
cudaError_t launch(cudaStream_t stream, Kernel kernel, long long grid, size_t smem, const KvQ4Attention& a, bool programmatic) {
    if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int HD, int NT, bool PAIR>
cudaError_t launch_spans(cudaStream_t stream, const KvQ4Attention& a) {
    constexpr size_t smem = (size_t)kWarps * kRing * q4_record(HD);
    static bool configured[kMaxDevices] = {false};   // function attributes are per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kvq4_span_kernel<HD, NT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    return launch(stream, kvq4_span_kernel<HD, NT, PAIR>, (long long)a.max_spans * a.sequences * a.kv_heads * a.col_blocks, smem, a, false);
}

template <int HD>
cudaError_t launch_hd(cudaStream_t stream, const KvQ4Attention& a) {
    constexpr int WIDE = HD == 256 ? 1 : 2;
    const bool pair = a.type == kQ4F32;
    cudaError_t e = a.span_cols == 8 ? (pair ? launch_spans<HD, 1, true>(stream, a) : launch_spans<HD, 1, false>(stream, a))
                                     : (pair ? launch_spans<HD, WIDE, true>(stream, a) : launch_spans<HD, WIDE, false>(stream, a));
    if (e == cudaSuccess && a.max_spans > 1) e = launch(stream, kvq4_merge_kernel<HD>, (long long)a.rows * a.q_heads, 0, a, true);
    return e;
}

}  // namespace

int kvq4_sm_count() {
    static int counts[kMaxDevices] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
    if (counts[dev] == 0 && (cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || counts[dev] <= 0)) counts[dev] = 148;
    return counts[dev];
}

namespace {

// Bytes of the spans' sums, and behind them room for the tile kernel's operands: at most kScratchMost, or what the sequences with
// enough rows can need.
constexpr size_t kScratchMost = 512u << 20;
size_t partial_bytes(const KvQ4Attention& a) {
    const size_t n = a.max_spans > 1 ? (size_t)a.rows * a.q_heads * a.max_spans * (a.head_dim + 2) * sizeof(float) : 0;
    return (n + 255) / 256 * 256;
}
int wanted_tiles(const KvQ4Attention& a) {
    const long long flats = (long long)a.rows * (a.q_heads / a.kv_heads);
    if ((long long)std::min(a.max_rows, a.rows) * (a.q_heads / a.kv_heads) <= a.tile_above) return 0;
    const long long keys = a.window > 0 ? std::min<long long>(a.max_keys, (long long)a.window + a.max_rows) : a.max_keys;
    const long long tiles = std::min<long long>(a.sequences, flats / (a.tile_above + 1)) * (keys / 128 + 2), room = (long long)(kScratchMost / ((size_t)512 * a.head_dim * a.kv_heads));
    return (int)std::min(tiles, room);
}

}  // namespace

size_t kvq4_workspace_bytes(const KvQ4Attention& args) {
    KvQ4Attention a = args;
    plan_spans(a);
    return partial_bytes(a) + (size_t)wanted_tiles(a) * 512 * a.head_dim * a.kv_heads;
}

cudaError_t launch_kvq4_attention(cudaStream_t stream, KvQ4Attention a) {
    if (a.rows <= 0 || a.sequences <= 0) return cudaSuccess;
    plan_spans(a);
    const size_t sums = partial_bytes(a);
    if (a.partial_bytes < sums) return cudaErrorInvalidValue;
    a.scratch = reinterpret_cast<unsigned char*>(a.partial) + sums;
    a.scratch_tiles = (int)std::min<size_t>((size_t)wanted_tiles(a), (a.partial_bytes - sums) / ((size_t)512 * a.head_dim * a.kv_heads));
    const int size = a.type == kQ4F32 ? 4 : 2;
    a.vector_q = aligned16(a.q, a.q_stride, size);
    a.vector_out = aligned16(a.out, a.out_stride, size);
    if ((long long)a.max_rows * (a.q_heads / a.kv_heads) > a.tile_above) {
        const cudaError_t e = launch_kvq4_tiles(stream, a);
        if (e != cudaSuccess) return e;
    }
    switch (a.head_dim) {
        case 64: return launch_hd<64>(stream, a);
        case 128: return launch_hd<128>(stream, a);
        case 256: return launch_hd<256>(stream, a);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace ribn
