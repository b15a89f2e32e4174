// Attention over the 4-bit paged KV cache (kvq4.cuh): a few query rows per sequence against long key ranges.
//
// The work is the list of all (sequence, kv head, block of columns) items' pages, one after the other (column = row of the sequence x
// query head of the group, up to 8 or 16 per block); every CTA has an equal run of it, whatever the sequences' lengths, so it begins
// and ends inside items; what it has of an item that it shares with others meets theirs in the merge kernel, in page order.  Within an
// item's run warp w of four takes pages w, w + 4, .. and is a pipeline of its own: page records come into its ring of shared memory
// by asynchronous copies, kRing - 1 pages ahead.  With m16n8k16 products, per page of 16 keys:
//   S^T = K Q^T   a masked nibble is a binary16 number by itself, code x 2^-24 (or, one nibble up, 2^-20: those dimensions' queries
//                 are held 2^-4 times), so a word of eight codes costs a shift and four masks and no conversion.  A group of 32
//                 dimensions is summed apart, beginning with -8 x the sum of its queries, and enters the score times its scale.
//                 Queries are scaled by a power of two per column, so that binary16 holds F16 and BF16 ones exactly.
//   O^T = V^T P^T a nibble under the exponent of 64 is 64 + code; one fused multiply-add with the scale and -72 x scale, both exact,
//                 gives the value.  P comes from the S^T layout by transposing 8 x 8 blocks across the warp.
// F32 queries and their probabilities are binary16 hi + lo pairs (two products each), K is converted as V is (the sums above begin
// far from where they end: 1.8e-6 off instead of 6e-7), and a page's sums are added in the registers, as an addition of the matrix
// instruction cuts at the sum's last bit.  Softmax in base 2; a column's reference moves only when a score passes it by 2^8, and P is
// held 2^7 times, so that small probabilities stay normal numbers.  F16 and BF16 rows have one binary16 for each, as a pair would take twice the
// products; they are divided by the sum of the rounded ones, so that a row's weights still add up to one.
// Against 64 bits F16 rows are then 1.0 to 1.3 times as far as the rounding of the result alone, with the sum of the unrounded ones up to 1.5 times.
// Results do not depend on where pages lie; how the work is cut, and with it the last bits, depends on the call's lengths.
//
// What bounds it: issuing.  A page takes a warp about 330 instructions, 96 of them on the logic pipe, which starts one every other
// clock, and three CTAs of four warps per SM issue two of three clocks: sixteen BF16 sequences of up to 32,768 keys, 32 / 8 heads, 395 MB,
// 97 us, 62 % of the copy bandwidth.  Short calls are a chain of memory's latencies: where the CTA's run begins, queries and page
// numbers, pages, and the merge's; one sequence of 1,024 keys takes 14 us with its append.  Tried: a grid of (span, item) instead of the
// list 142 us for the sixteen, four CTAs per SM with 48 bytes of spills 103; for up to 16 columns three CTAs instead of two, 290 bytes of
// spills, 175 against 166 us (40 sequences of four rows, windows of 4,096 keys), and blocks of 8 columns 189.
#include <math.h>

#include <algorithm>

#include "kvq4.cuh"

namespace ribn {

namespace {

constexpr int kWarps = 4;
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
// 64 + the nibbles of bits 4 .. 7 of both halves, times the scale, minus 72 times it
__device__ __forceinline__ uint32_t value(uint32_t x, __half2 scale, __half2 minus72) {
    return bits_of(__hfma2(half2_of(and_or(x, 0x00F000F0u, 0x54005400u)), scale, minus72));
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

// A sequence in the list of work.  Its row i is at position base + i.
struct Sequence {
    int row0, n, base;
    int page0, pages;      // that some row sees
    int blocks;            // of columns
    int set_up;            // see plan_spans
    // of an item, in pages; one without keys writes its zeros
    __device__ __forceinline__ int length() const { return pages > 0 ? pages + set_up : 1; }
    __device__ __forceinline__ long long weight(int kv_heads) const { return (long long)kv_heads * blocks * length(); }
};
__device__ __forceinline__ Sequence sequence_of(const KvQ4Attention& a, int s) {
    Sequence q;
    const int group = a.q_heads / a.kv_heads;
    q.row0 = max(a.cu_rows[s], 0);
    q.n = max(0, min(a.cu_rows[s + 1], a.rows) - q.row0);
    q.base = min(max(a.lengths[s], 0), a.pages_per_sequence * kQ4Page) - q.n;
    const int high = max(0, q.base + q.n), low = a.window > 0 ? max(0, q.base - a.window + 1) : 0;
    q.page0 = low / kQ4Page;
    q.set_up = a.set_up;
    q.pages = high > low ? (high + kQ4Page - 1) / kQ4Page - q.page0 : 0;
    const long long cols = (long long)min(q.n, a.max_rows) * group;
    q.blocks = cols > a.tile_above ? 0 : (int)((cols + a.span_cols - 1) / a.span_cols);   // 0: the tile kernel's
    return q;
}
// Pages per CTA of a list of `total`: whole rounds of the four warps
__device__ __forceinline__ long long share_of(const KvQ4Attention& a, long long total) {
    const long long even = (total + a.grid - 1) / a.grid;
    return (max(even, (long long)kWarps) + kWarps - 1) / kWarps * kWarps;
}
// One item's columns
struct Block {
    int cols, flat0, first_row, last_row;
    int low, high;         // keys that some row of the block sees: low <= key < high
};
__device__ __forceinline__ Block block_of(const KvQ4Attention& a, const Sequence& q, int cb) {
    Block b;
    const int group = a.q_heads / a.kv_heads;
    b.flat0 = cb * a.span_cols;
    b.cols = min(a.span_cols, min(q.n, a.max_rows) * group - b.flat0);
    b.first_row = b.flat0 / group;
    b.last_row = (b.flat0 + b.cols - 1) / group;
    b.high = max(0, q.base + b.last_row + 1);
    b.low = a.window > 0 ? max(0, q.base + b.first_row - a.window + 1) : 0;
    return b;
}

constexpr int kRing = 4;   // page records per warp: one read, three on their way
// F32 rows: a thread's sums move to shared memory after so many pages.  In one place, thousands of keys of 2^-25 of the largest fell below the sums'
// last bits (one row, 60,000 keys of which three have all but 5e-4, one CTA: 3.8e-5 off, so less than 4e-6).
constexpr int kKept = 32;
template <int HD, int NT, bool PAIR>
constexpr size_t kSpanSmem = (size_t)kWarps * kRing * q4_record(HD) + (PAIR ? kWarps * 32 * (2 + HD / 4) * NT * sizeof(float) : 0);

// NT: column tiles of 8.  PAIR: F32 queries.
template <int HD, int NT, bool PAIR>
__global__ void __launch_bounds__(kWarps * 32, HD <= 128 && NT == 1 ? 3 : 2) kvq4_span_kernel(const KvQ4Attention a) {
    constexpr int NG = HD / 32, WORDS = NG < 4 ? NG : 4, SUB = NG / WORDS;
    constexpr int RECORD = q4_record(HD), RING = kRing, REC = HD + 2;
    constexpr int BLOCK = kQ4Page * 16 * WORDS;   // bytes of codes of one sub
    extern __shared__ __align__(128) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.q_heads / a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- where this CTA's run begins: the list's length before each sequence, a stretch of sequences per thread
    __shared__ long long sums[kWarps];
    __shared__ long long at_sequence_before;
    __shared__ int at_sequence;
    const int stretch = (a.sequences + kWarps * 32 - 1) / (kWarps * 32), s0 = min(a.sequences, (int)threadIdx.x * stretch), s1 = min(a.sequences, s0 + stretch);
    long long mine_sum = 0;
    for (int i = s0; i < s1; ++i) mine_sum += sequence_of(a, i).weight(a.kv_heads);
    long long upto = mine_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long total = 0, before = upto - mine_sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    const long long share = share_of(a, total);
    long long at = blockIdx.x * share;
    const long long stop = min(total, at + share);
    if (blockIdx.x == 0 && a.grid > 1) {   // for the merge: an item may have runs in several CTAs
        long long x = before;
        for (int i = s0; i < s1; ++i) { a.prefix[i] = x; x += sequence_of(a, i).weight(a.kv_heads); }
        if (threadIdx.x == 0) a.prefix[a.sequences] = total;
    }
    if (at >= stop) return;
    if (before <= at && at < before + mine_sum) {
        long long x = before;
        int i = s0;
        for (;; ++i) {
            const long long w = sequence_of(a, i).weight(a.kv_heads);
            if (at < x + w) break;
            x += w;
        }
        at_sequence = i;
        at_sequence_before = x;
    }
    __syncthreads();
    int s = at_sequence;
    long long s_before = at_sequence_before;
    Sequence seq = sequence_of(a, s);
    for (bool first_run = true; at < stop; first_run = false) {
    while (at >= s_before + seq.weight(a.kv_heads)) {   // the next sequence that has work (`at` is inside of the list)
        s_before += seq.weight(a.kv_heads);
        seq = sequence_of(a, ++s);
    }
    const long long inside = at - s_before;
    const int item = (int)(inside / seq.length()), offset = (int)(inside - (long long)item * seq.length());
    const int kvh = item / seq.blocks, cb = item % seq.blocks, run = (int)min((long long)(seq.length() - offset), stop - at);
    const bool whole = run == seq.length();
    const Block b = block_of(a, seq, cb);
    // the run's pages, those that the block sees
    const int begin = max(seq.page0 + max(offset - seq.set_up, 0), b.low / kQ4Page);
    const int end = max(begin, min(seq.page0 + max(min(offset + run - seq.set_up, seq.pages), 0), (b.high + kQ4Page - 1) / kQ4Page));
    at += run;
    if (begin == end) {   // none: zeros, or a share of the item that counts for nothing
        for (int i = threadIdx.x; i < b.cols * REC; i += kWarps * 32) {
            const int col = i / REC, d = i % REC, flat = b.flat0 + col;
            if (!whole) a.partial[((2ll * blockIdx.x + (first_run ? 0 : 1)) * a.span_cols + col) * REC + d] = d == HD ? -INFINITY : 0.0f;
            else if (d < HD) store_value(a, (seq.row0 + flat / group) * a.out_stride + (long long)(kvh * group + flat % group) * HD + d, 0.0f);
        }
        continue;
    }
    const int mine = max(0, (end - begin - warp + kWarps - 1) / kWarps);   // this warp's pages
    const int32_t* table = a.page_tables + s * a.table_stride + begin + warp;
    const uint32_t ring = smem_at(smem) + warp * (RING * RECORD);
    const unsigned char* head = a.cache + (long long)kvh * RECORD;
    const long long page_stride = (long long)a.kv_heads * RECORD;

    // the columns' queries, asked for before what the pages' addresses wait for
    uint32_t raw[NT][NG][PAIR ? 8 : 4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + g, flat = b.flat0 + col;
#pragma unroll
        for (int G = 0; G < NG; ++G) {
#pragma unroll
            for (int i = 0; i < (PAIR ? 8 : 4); ++i) raw[nt][G][i] = 0u;
            if (col < b.cols) q4_load_raw(a.q, (seq.row0 + flat / group) * a.q_stride + (long long)(kvh * group + flat % group) * HD + 32 * G + 8 * t, a.vector_q, raw[nt][G]);
        }
    }
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

    // B fragments of Q^T: column 8 nt + g; of group G the dimensions 32 G + 8 t + {0, 4, 2, 6} and, 2^-4 times (not PAIR), {1, 5, 3, 7}
    uint32_t qh[NT][NG][4], ql[NT][PAIR ? NG : 1][4];
    float start[NT][PAIR ? 1 : NG][2], factor[NT][2];
    int last[NT][2], lowest[NT][2];   // keys that columns 8 nt + 2 t + {0, 1} see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float x[NG][8], top = 0.0f;
#pragma unroll
        for (int G = 0; G < NG; ++G) {
            q4_values(raw[nt][G], a.type, x[G]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[G][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e brings the largest to [2^13, 2^14)
        const int e = top > 0.0f && top < INFINITY ? max(-126, min(126, 140 - (int)(__float_as_uint(top) >> 23))) : 0;
        const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
        const float f = copysignf(q4_factor(down * fabsf(a.scale)), a.scale) * (PAIR ? 1.0f : 16777216.0f);   // (codes are held 2^-24 times)
        factor[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
        factor[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int G = 0; G < NG; ++G) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[G][i] *= up; sum += x[G][i]; }
            if constexpr (!PAIR) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= -8.0f / 16777216.0f;
                start[nt][G][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                start[nt][G][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = (u & 1) * 2 + (u >> 1);   // 0, 2, 1, 3: the word's pairs are (i, i + 4)
                const float m = !PAIR && (u >> 1) ? 0.0625f : 1.0f;
                const __half2 h = __floats2half2_rn(x[G][i] * m, x[G][i + 4] * m);
                qh[nt][G][u] = bits_of(h);
                if (PAIR) {
                    const float2 back = __half22float2(h);
                    ql[nt][PAIR ? G : 0][u] = bits_of(__floats2half2_rn(x[G][i] * m - back.x, x[G][i + 4] * m - back.y));
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int column = nt * 8 + 2 * t + c;
            last[nt][c] = column < b.cols ? seq.base + (b.flat0 + column) / group : -1;
            lowest[nt][c] = a.window > 0 ? last[nt][c] - a.window + 1 : 0;
        }
    }
    // keys that every column sees
    const int all_low = a.window > 0 ? seq.base + b.last_row - a.window + 1 : 0, all_high = seq.base + b.first_row;

    float o[NT][2 * NG][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < 2 * NG; ++mt) { o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f; }
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.0f;
    }
    // PAIR, of each column tile: where l and o are kept, kWarps * 32 floats apart
    const bool keeps = PAIR && mine > kKept;
    float* const kept = reinterpret_cast<float*>(smem + kWarps * RING * RECORD) + threadIdx.x;
    constexpr int KEPT = (2 + 8 * NG) * kWarps * 32;
    auto keep = [&](bool first) {   // the sums so far, and from zero on
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int u = 0; u < 2 + 8 * NG; ++u) {
                float& x = u < 2 ? l[nt][u & 1] : o[nt][(u - 2) >> 2 & (2 * NG - 1)][(u - 2) & 3];
                float* const to = kept + nt * KEPT + u * kWarps * 32;
                *to = first ? x : *to + x;
                x = 0.0f;
            }
        }
    };

    for (int i = 0; i < mine; ++i) {
        issue(i + RING - 1);
        if (PAIR && i > 0 && i % kKept == 0) keep(i == kKept);
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
                    if constexpr (PAIR) {
                        const __half2 minus72 = __float2half2_rn(-72.0f);
                        const __half2 k0 = half2_of(__byte_perm(s0[G >> 1], 0u, (G & 1) ? 0x3232u : 0x1010u)), k1 = half2_of(__byte_perm(s1[G >> 1], 0u, (G & 1) ? 0x3232u : 0x1010u));
                        const __half2 z0 = __hmul2(k0, minus72), z1 = __hmul2(k1, minus72);
                        const uint32_t even[4] = {value(w0[w] * 16u, k0, z0), value(w1[w] * 16u, k1, z1), value(x0 * 16u, k0, z0), value(x1 * 16u, k1, z1)};
                        const uint32_t odd[4] = {value(w0[w], k0, z0), value(w1[w], k1, z1), value(x0, k0, z0), value(x1, k1, z1)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma(acc, even, ql[nt][G][0], ql[nt][G][1], acc);
                            mma(acc, odd, ql[nt][G][2], ql[nt][G][3], acc);
                            mma(acc, even, qh[nt][G][0], qh[nt][G][1], acc);
                            mma(acc, odd, qh[nt][G][2], qh[nt][G][3], acc);
#pragma unroll
                            for (int u = 0; u < 4; ++u) sc[nt][u] += acc[u];
                        }
                    } else {
                        const uint32_t even[4] = {w0[w] & 0x000F000Fu, w1[w] & 0x000F000Fu, x0 & 0x000F000Fu, x1 & 0x000F000Fu};
                        const uint32_t odd[4] = {w0[w] & 0x00F000F0u, w1[w] & 0x00F000F0u, x0 & 0x00F000F0u, x1 & 0x00F000F0u};
                        const float2 k0 = __half22float2(half2_of(s0[G >> 1])), k1 = __half22float2(half2_of(s1[G >> 1]));
                        const float f0 = (G & 1) ? k0.y : k0.x, f1 = (G & 1) ? k1.y : k1.x;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float from[4] = {start[nt][G][0], start[nt][G][1], start[nt][G][0], start[nt][G][1]};
                            float acc[4];
                            mma(acc, even, qh[nt][G][0], qh[nt][G][1], from);
                            mma(acc, odd, qh[nt][G][2], qh[nt][G][3], acc);
                            sc[nt][0] = fmaf(acc[0], f0, sc[nt][0]); sc[nt][1] = fmaf(acc[1], f0, sc[nt][1]);
                            sc[nt][2] = fmaf(acc[2], f1, sc[nt][2]); sc[nt][3] = fmaf(acc[3], f1, sc[nt][3]);
                        }
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
                if (PAIR && i >= kKept) {
#pragma unroll 4
                    for (int u = 0; u < 2 + 8 * NG; ++u) kept[nt * KEPT + u * kWarps * 32] *= f[u & 1];
                }
            }
        }
        uint32_t ph[NT][2], pl[PAIR ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float m0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0] - kHeld, m1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1] - kHeld;
            const float p0 = exp2_approx(sc[nt][0] - m0), p1 = exp2_approx(sc[nt][1] - m1), p2 = exp2_approx(sc[nt][2] - m0), p3 = exp2_approx(sc[nt][3] - m1);
            const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
            if constexpr (PAIR) {
                l[nt][0] += p0 + p2; l[nt][1] += p1 + p3;
            } else {
                const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                l[nt][0] += b0.x + b1.x; l[nt][1] += b0.y + b1.y;
            }
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
                    const uint32_t u0 = w0[w] >> 8, u1 = w1[w] >> 8;   // (to the left by a multiplication, which runs beside the logic)
                    const uint32_t lower[4] = {value(w0[w] * 16u, a0, b0), value(w0[w], a0, b0), value(w1[w] * 16u, a1, b1), value(w1[w], a1, b1)};
                    const uint32_t upper[4] = {value(u0 * 16u, a0, b0), value(u0, a0, b0), value(u1 * 16u, a1, b1), value(u1, a1, b1)};
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
    if (keeps) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int u = 0; u < 2 + 8 * NG; ++u) (u < 2 ? l[nt][u & 1] : o[nt][(u - 2) >> 2 & (2 * NG - 1)][(u - 2) & 3]) += kept[nt * KEPT + u * kWarps * 32];
        }
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
    const int live = min(kWarps, end - begin);   // warps that have pages
    const float* recs = reinterpret_cast<const float*>(smem);
    for (int col = warp; col < b.cols; col += kWarps) {
        const int flat = b.flat0 + col, row = seq.row0 + flat / group, qh_index = kvh * group + flat % group;
        float top = -INFINITY;
        for (int w = 0; w < live; ++w) top = fmaxf(top, recs[w * kWarpFloats + col * REC + HD]);
        float acc[HD / 32], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
        for (int w = 0; w < live; ++w) {
            const float mw = recs[w * kWarpFloats + col * REC + HD], fw = mw == -INFINITY ? 0.0f : exp2_approx(mw - top);
            sum = fmaf(recs[w * kWarpFloats + col * REC + HD + 1], fw, sum);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(recs[w * kWarpFloats + col * REC + lane + 32 * i], fw, acc[i]);
        }
        if (whole) {
            const long long to = row * a.out_stride + (long long)qh_index * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) store_value(a, to + lane + 32 * i, sum > 0.0f || sum != sum ? acc[i] / sum : 0.0f);
        } else {   // the CTA's first run in its first place, its last in the second: those between are whole items
            float* pp = a.partial + ((2ll * blockIdx.x + (first_run ? 0 : 1)) * a.span_cols + col) * REC;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) pp[lane + 32 * i] = acc[i];
            if (lane == 0) { pp[HD] = top; pp[HD + 1] = sum; }
        }
    }
    __syncthreads();   // the rings are free again
    }
}

// out = sum_r acc_r 2^(m_r - M) / sum_r l_r 2^(m_r - M) over an item's runs: four warps per (item, column), warp w runs w, w + 4, ..,
// then the warps in order.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) kvq4_merge_kernel(const KvQ4Attention a) {
    constexpr int DPL = HD / 32, REC = HD + 2, GROUP = 4;
    __shared__ float sums[kWarps][HD + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.q_heads / a.kv_heads;
    int id = blockIdx.x;
    const int col = id % a.merge_cols; id /= a.merge_cols;
    const int cb = id % a.col_blocks; id /= a.col_blocks;
    const int kvh = id % a.kv_heads, s = id / a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Sequence q = sequence_of(a, s);
    if (cb >= q.blocks) return;
    const Block b = block_of(a, q, cb);
    if (col >= b.cols) return;
    const long long share = share_of(a, __ldcg(a.prefix + a.sequences)), from = __ldcg(a.prefix + s) + (long long)(kvh * q.blocks + cb) * q.length();
    const int c0 = (int)(from / share), runs = (int)((from + q.length() - 1) / share) - c0 + 1;
    if (runs <= 1) return;   // written by the span kernel
    // the item's run in CTA c0 is that one's last, in the others their first
    const bool last_of_c0 = from > c0 * share;
    auto record = [&](int r) { return a.partial + ((2ll * (c0 + r) + (r == 0 && last_of_c0 ? 1 : 0)) * a.span_cols + col) * REC; };
    float top = -INFINITY;
    for (int r = lane; r < runs; r += 32) top = fmaxf(top, __ldcg(record(r) + HD));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum[DPL], denom = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) sum[i] = 0.0f;
    for (int r0 = warp; r0 < runs; r0 += kWarps * GROUP) {
        float v[GROUP][DPL], mx[GROUP], lx[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const int r = r0 + kWarps * u;
            const float* rec = record(min(r, runs - 1));
#pragma unroll
            for (int i = 0; i < DPL; ++i) v[u][i] = __ldcg(rec + lane + 32 * i);
            mx[u] = r < runs ? __ldcg(rec + HD) : -INFINITY;
            lx[u] = __ldcg(rec + HD + 1);
        }
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const float w = mx[u] == -INFINITY ? 0.0f : exp2_approx(mx[u] - top);   // past the last run, without keys, or lost in NaN (which 0 x keeps)
            denom = fmaf(lx[u], w, denom);
#pragma unroll
            for (int i = 0; i < DPL; ++i) sum[i] = fmaf(v[u][i], w, sum[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < DPL; ++i) sums[warp][lane + 32 * i] = sum[i];
    if (lane == 0) sums[warp][HD] = denom;
    __syncthreads();
    const float all = ((sums[0][HD] + sums[1][HD]) + sums[2][HD]) + sums[3][HD];
    const int flat = b.flat0 + col;
    const long long to = (q.row0 + flat / group) * a.out_stride + (long long)(kvh * group + flat % group) * HD;
    for (int d = threadIdx.x; d < HD; d += kWarps * 32) {
        const float value = ((sums[0][d] + sums[1][d]) + sums[2][d]) + sums[3][d];
        store_value(a, to + d, all > 0.0f || all != all ? value / all : 0.0f);
    }
}

bool aligned16(const void* p, long long stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; }

// Columns per CTA, and how many CTAs share the list.
void plan_spans(KvQ4Attention& a) {
    const int group = a.q_heads / a.kv_heads;
    // More columns take the tensor-memory kernel: eight BF16 sequences of 2,000 keys with 64 columns 55 us here and 80 there, with 128 91 and
    // 66.  (Heads of 256 have no such kernel: two tiles' sums would take all of tensor memory;
    // one tile a CTA would fit and was not built.)
    a.tile_above = a.head_dim == 256 ? 0x7fffffff : 64;
    const int cols = (int)std::min<long long>((long long)std::min(a.max_rows, a.rows) * group, a.tile_above);
    // 16 columns share a page's conversion; with heads of 256 their sums do not fit in the registers (1,080 bytes of spills)
    a.span_cols = cols <= 8 || a.head_dim == 256 ? 8 : 16;
    a.col_blocks = (cols + a.span_cols - 1) / a.span_cols;
    a.merge_cols = std::min(cols, a.span_cols);
    // An item's set-up and fold, a chain of memory's latencies, count as this many pages.  (As 8, CTAs with many short items were the last
    // ones by far.)  16 columns, 40 sequences of four rows behind windows of 4,096 keys, a tenth of them with four keys: as 20 220 us, 40
    // 165, 64 159, but 64 even sequences of 4,096 keys as 40 138 and as 64 142.  8 columns, 64 sequences of up to 1,500 keys: as 20 45.9,
    // 40 47.0, 64 47.4; sixteen of up to 32,768: 98.6, 100.5, 102.5.
    a.set_up = a.span_cols == 8 ? 20 : 40;
    const long long keys = a.window > 0 ? std::min<long long>(a.max_keys, (long long)a.window + a.max_rows + kQ4Page) : a.max_keys;
    const long long pages = std::max(1ll, (keys + kQ4Page - 1) / kQ4Page), items = (long long)a.sequences * a.kv_heads * a.col_blocks;
    const long long resident = (long long)a.sms * (a.head_dim <= 128 && a.span_cols == 8 ? 3 : 2);   // as their launch bounds say
    a.grid = (int)std::max(1ll, std::min(resident, (items * pages + kWarps - 1) / kWarps));
}

template <typename Kernel>
cudaError_t launch(cudaStream_t stream, Kernel kernel, long long grid, size_t smem, const KvQ4Attention& a) {
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
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int HD, int NT, bool PAIR>
cudaError_t launch_spans(cudaStream_t stream, const KvQ4Attention& a) {
    constexpr size_t smem = kSpanSmem<HD, NT, PAIR>;
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
    return launch(stream, kvq4_span_kernel<HD, NT, PAIR>, a.grid, smem, a);
}

template <int HD>
cudaError_t launch_hd(cudaStream_t stream, const KvQ4Attention& a) {
    constexpr int WIDE = HD == 256 ? 1 : 2;
    const bool pair = a.type == kQ4F32;
    cudaError_t e = a.span_cols == 8 ? (pair ? launch_spans<HD, 1, true>(stream, a) : launch_spans<HD, 1, false>(stream, a))
                                     : (pair ? launch_spans<HD, WIDE, true>(stream, a) : launch_spans<HD, WIDE, false>(stream, a));
    if (e == cudaSuccess && a.grid > 1) e = launch(stream, kvq4_merge_kernel<HD>, (long long)a.sequences * a.kv_heads * a.col_blocks * a.merge_cols, 0, a);
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
size_t prefix_bytes(const KvQ4Attention& a) { return ((size_t)a.sequences + 1) * sizeof(long long); }
size_t partial_bytes(const KvQ4Attention& a) {
    const size_t n = a.grid > 1 ? prefix_bytes(a) + (size_t)a.grid * 2 * a.span_cols * (a.head_dim + 2) * sizeof(float) : 0;
    return (n + 255) / 256 * 256;
}
bool has_tiles(const KvQ4Attention& a) { return (long long)std::min(a.max_rows, a.rows) * (a.q_heads / a.kv_heads) > a.tile_above; }
long long seen_keys(const KvQ4Attention& a) { return a.window > 0 ? std::min<long long>(a.max_keys, (long long)a.window + a.max_rows) : a.max_keys; }
int wanted_tiles(const KvQ4Attention& a) {
    if (!has_tiles(a)) return 0;
    const long long flats = (long long)a.rows * (a.q_heads / a.kv_heads);
    const long long tiles = std::min<long long>(a.sequences, flats / (a.tile_above + 1)) * (seen_keys(a) / 128 + 2), room = (long long)(kScratchMost / ((size_t)512 * a.head_dim * a.kv_heads));
    return (int)std::min(tiles, room);
}
// While query tiles leave SMs idle their keys are shared, two key tiles to a CTA at least: 16 rows behind 8,000 keys, 32 / 8 heads, 182 us
// without.  The sums of rows x q_heads x splits are those of at most 256 rows per SM.
// Long ranges are shared whatever the SMs: a sum in tensor memory is cut at its last bit by every product of 16 keys and comes out about 0.8 x 2^-24
// smaller for each (F32 rows fold theirs): F16 rows behind 131,072 keys 3.9e-4 with all of them in one CTA, beside roundings of 2.3e-4, and less than
// 1.2e-4 with 32,768.  While the sums take at most kSumsMost.  2,048 BF16 rows behind 65,536 keys, 32 / 8 heads: 2.02 ms before, 2.07
// so; behind 131,072: 4.08 and 3.92.
constexpr long long kLongest = 32768 / 128;
constexpr size_t kSumsMost = 256u << 20;
size_t sums_of(const KvQ4Attention& a) { return (size_t)a.rows * a.q_heads * (a.head_dim + 4) * sizeof(float); }
int wanted_splits(const KvQ4Attention& a) {
    if (!has_tiles(a)) return 1;
    const long long ctas = std::max(1ll, kvq4_tile_places(a) * a.kv_heads), tiles = std::max(1ll, seen_keys(a) / 128 + 1);
    const long long idle = std::max(1ll, std::min(a.sms / ctas, (tiles + 1) / 2));
    const long long exact = a.type == kQ4F32 ? 1 : std::min((tiles + kLongest - 2) / kLongest, (long long)(kSumsMost / sums_of(a)));
    return (int)std::max(idle, exact);
}
size_t split_bytes(const KvQ4Attention& a) {
    const int splits = wanted_splits(a);
    return splits > 1 ? splits * sums_of(a) : 0;
}

}  // namespace

int kvq4_most_sms() {
    int count = 0, most = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess) count = 0;
    for (int dev = 0; dev < count; ++dev) {
        int sms = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) most = std::max(most, sms);
    }
    return most > 0 ? most : 148;
}

size_t kvq4_workspace_bytes(const KvQ4Attention& args, int sms) {
    KvQ4Attention a = args;
    a.sms = sms;
    plan_spans(a);
    return partial_bytes(a) + split_bytes(a) + (size_t)wanted_tiles(a) * 512 * a.head_dim * a.kv_heads;
}

cudaError_t launch_kvq4_attention(cudaStream_t stream, KvQ4Attention a) {
    if (a.rows <= 0 || a.sequences <= 0) return cudaSuccess;
    a.sms = kvq4_sm_count();
    plan_spans(a);
    const size_t runs = partial_bytes(a), sums = runs + split_bytes(a);
    if (a.partial_bytes < sums) return cudaErrorInvalidValue;
    a.tile_splits = wanted_splits(a);
    unsigned char* scratch = reinterpret_cast<unsigned char*>(a.partial);
    a.prefix = reinterpret_cast<long long*>(scratch);
    a.partial = reinterpret_cast<float*>(scratch + prefix_bytes(a));
    a.tile_partial = reinterpret_cast<float*>(scratch + runs);
    a.scratch = scratch + sums;
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
