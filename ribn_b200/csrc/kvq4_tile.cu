// Attention of many query rows per sequence over the 4-bit paged KV cache (kvq4.cuh) on the tcgen05 tensor cores.
//
// A CTA serves one (sequence, kv head) and two tiles of 128 query rows (row = row of the sequence x query head of the group), each
// with softmax warps of its own, so that one tile's products run while the other's probabilities are formed.  Per 128 keys:
//   S = Q K^T   A = the queries as binary16 in shared memory, scaled by a power of two per row, B = K;
//   P           two threads own a row, 64 keys each: softmax in base 2 against a reference that moves only when a score passes it by
//               2^8, P (held 2^7 times, so that small ones stay normal numbers) as binary16 over S in tensor memory, divided at the end by
//               the sum of the rounded ones, so that a row's weights add up to one (1.1 % of the time; a row of one key has its value);
//   O += P V    A = P from tensor memory, B = V^T.
// K and V^T come as operands: from memory, where kvq4_expand_kernel has left them, once for all query rows of a call, or, where the
// call has no room for that, from seven warps that turn page records into them.  A nibble under the exponent of 64 is 64 + code; one
// fused multiply-add with the scale and -72 x scale, both exact, gives the value.  Sums over dimensions and keys may run in any order, so
// neither operand is reordered: of K the word's pairs (i, i + 4) stay neighbours and the queries' dimensions follow, of V a lane's keys
// 2 t, 2 t + 1, 2 t + 8, 2 t + 9 stay neighbours and the rows of K follow.
// F32 queries and probabilities are binary16 hi + lo pairs, two products each, and a row has one thread; as an addition in tensor
// memory cuts at the sum's last bit, their sums over 256 keys move into the rows' registers.
// Roles of the 24 warps (16 of F32 rows): softmax and output of tile 0 and 1, four K, one issues the products, three V.  Every wait is
// bounded; where one runs out the CTA's rows become NaN, and what it has in flight is waited for (with a limit too) before it ends.
//
// What bounds it: a tile's chain.  Its products take 1,024 clocks, its scores 1,300 to 1,600 to become probabilities (exponentials: 16 a
// clock per SM, a quarter of them moved to the multiply-add pipe), and handing over costs about 700 each time, while the other tile's
// products fill 1,024 of that.  2,048 BF16 rows behind 14,336 keys, 32 / 8 heads: 555 us in a replayed graph with their append, 16 us of
// expansion and cold inputs, 928 TFLOP/s (256 CTAs on 148 SMs: the second turn fills 73 % of them).  Tried, of the kernel when it took 520: conversion by seven warps beside it 585; one
// thread per row 545 (its instructions wait for one another); one vote per 128 scores, with spills, 720; a warp per tile for the
// products 565 (both tiles' products then run at the same time, and both softmaxes); no exponentials by the polynomial 553.
// Short chunks are latencies and instructions fetched for the first time: 777 F32 rows of 16 / 8 heads 51 us with append and merges.
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

#include "kvq4.cuh"
#include "tmem.cuh"

namespace ribn {

namespace {

constexpr int kRows = 128, kKeys = 128, kKWarps = 4, kVWarps = 3;
constexpr int kTilePages = kKeys / kQ4Page;
constexpr uint32_t kLandPolls = 1u << 14;   // a poll that fails takes 4 us: 65 ms for a copy to land
constexpr float kHeld = 7.0f, kSlack = 8.0f;
constexpr int kPolynomial = 4;   // of 16 pairs of probabilities: those whose exponentials the multiply-add pipe computes
constexpr float kUnset = -3e38f;   // below every finite score's place
// PAIR: shares of the 512 x 128 registers at launch, 256 x (192 + 64).  (The other form keeps its 768 x 80.)
constexpr int kSoftmaxRegs = 192, kOtherRegs = 64;
constexpr int kWindow = 2;   // PAIR: key tiles whose products one sum in tensor memory holds

template <int HD, bool PAIR>
struct Tile {
    static constexpr int PIECES = HD / 8;                         // 16-byte pieces of a query or key row
    static constexpr int Q_STRIDE = kRows * 16, Q_TILE = PIECES * Q_STRIDE;
    static constexpr int K_STRIDE = kKeys * 16, K_TILE = PIECES * K_STRIDE;
    static constexpr int V_STRIDE = HD * 16, V_TILE = kKeys / 8 * V_STRIDE;
    static constexpr int PLANES = PAIR ? 2 : 1, K_SLOTS = 2, V_SLOTS = PAIR ? 1 : 2;
    static constexpr int K_AT = 2 * PLANES * Q_TILE, V_AT = K_AT + K_SLOTS * K_TILE, BARS = V_AT + V_SLOTS * V_TILE;
    static constexpr int FACTORS = BARS + 192, XCH = FACTORS + (PAIR ? 0 : 2 * kRows * 4);
    static constexpr size_t SMEM = XCH + (PAIR ? 0 : 4 * kRows * 4);
    // threads that share a query row's keys
    static constexpr int HALVES = PAIR ? 1 : 2;
    static constexpr int K_WARP = 8 * HALVES, MMA_WARP = K_WARP + kKWarps, V_WARP = MMA_WARP + 1, THREADS = (V_WARP + kVWarps) * 32;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
          "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_tie32(float (&v)[32]) {   // the values of a load, after its wait
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]) :: "memory");
    }
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of a pair on the multiply-add pipe, whose instructions take two values each, beside the sixteen a clock of the special function
// unit: x = n + f, n the nearest integer (left in the low bits of x + 3 x 2^22), 2^f by the polynomial of degree 3 that is nearest in
// relative error over [-1/2, 1/2] (7.5e-5, found by Remez's exchange; binary16 is off by up to 4.9e-4), n added to the exponent.  NaN does
// not pass (it comes out as 2^-126): rows whose queries are not finite become NaN by their flag.
__device__ __forceinline__ float2 exp2_pair(float2 x) {
    constexpr float kMagic = 12582912.0f;
    x = make_float2(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f));
    const float2 r = __fadd2_rn(x, make_float2(kMagic, kMagic));
    const float2 f = __fadd2_rn(x, __ffma2_rn(r, make_float2(-1.0f, -1.0f), make_float2(kMagic, kMagic)));
    float2 p = __ffma2_rn(make_float2(0.0551716685f, 0.0551716685f), f, make_float2(0.242611125f, 0.242611125f));
    p = __ffma2_rn(p, f, make_float2(0.693260968f, 0.693260968f));
    p = __ffma2_rn(p, f, make_float2(0.999928057f, 0.999928057f));
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}
// 2^k, k in [-126, 127]
__device__ __forceinline__ float power2(int k) { return __int_as_float((k + 127) << 23); }
// x0, x1 = hi + lo as binary16 pairs
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 back = __half22float2(h), rest = __fadd2_rn(make_float2(x0, x1), make_float2(-back.x, -back.y));
    hi = as_bits(h);
    lo = as_bits(__floats2half2_rn(rest.x, rest.y));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
template <int WORDS>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 1) {
        w[0] = __ldg(reinterpret_cast<const unsigned int*>(p));
    } else if constexpr (WORDS == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x; w[1] = v.y;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
}
// The four value pairs of a word: nibbles (i, i + 4), i = 0..3.  Shifts to the left are multiplications, which run beside the logic.
__device__ __forceinline__ void word_values(uint32_t w, __half2 s, __half2 minus72, uint32_t (&y)[4]) {
    const uint32_t up = w >> 8;
    const uint32_t x[4] = {w * 16u, w, up * 16u, up};
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = as_bits(__hfma2(as_half2(and_or(x[i], 0x00F000F0u, 0x54005400u)), s, minus72));
}
__device__ __forceinline__ float most_of(const float (&s)[32]) {
    float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int u = 4; u < 32; u += 4) {
#pragma unroll
        for (int v = 0; v < 4; ++v) top[v] = fmaxf(top[v], s[u + v]);
    }
    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// A column of a key tile holds key (column & ~15) + key_of_place(column & 15)
__device__ __forceinline__ constexpr int key_of_place(int p) { return 2 * (p >> 2) + (p & 1) + 8 * ((p >> 1) & 1); }

// Where a sequence's key tiles lie among those of all sequences of this kernel: [first, first + count) from key tile `tile0` on.
struct Tiles {
    int first, count, tile0;
};
__device__ __forceinline__ int tiles_of(const KvQ4Attention& a, int s, int& tile0, int& low, int& high) {
    const int group = a.q_heads / a.kv_heads, begin = a.cu_rows[s], end = a.cu_rows[s + 1], length = a.lengths[s];
    const int row0 = max(begin, 0), all = min(end, a.rows) - row0, n = min(all, a.max_rows);
    tile0 = low = high = 0;
    if (n <= 0 || (long long)n * group <= a.tile_above) return 0;
    const int base = min(max(length, 0), a.pages_per_sequence * kQ4Page) - all;
    high = max(0, base + n);
    low = a.window > 0 ? max(0, base - a.window + 1) : 0;
    tile0 = low / kKeys;
    return max(0, (high + kKeys - 1) / kKeys - tile0);
}
__device__ __forceinline__ Tiles tiles_before(const KvQ4Attention& a, int s, int lane) {   // by a whole warp
    int before = 0;
    for (int i = lane; i < s; i += 32) {
        int tile0, low, high;
        before = min(before + tiles_of(a, i, tile0, low, high), 1 << 20);   // (more than any scratch has; 32 such sums fit in the word)
    }
    Tiles r;
    r.first = __reduce_add_sync(0xffffffffu, before);
    int low, high;   // keys that some row sees
    r.count = tiles_of(a, s, r.tile0, low, high);
    return r;
}

// The pair of query tiles of this CTA: sequences in order, each one's later rows, which have the most keys, first.
struct Work {
    int s, row0, n, base, flat0;   // flat0: first query row of tile 0
};
__device__ __forceinline__ bool find_work(const KvQ4Attention& a, int place, int lane, Work& w) {
    const int group = a.q_heads / a.kv_heads;
    for (int s0 = 0; s0 < a.sequences; s0 += 32) {
        const int s = s0 + lane;
        int n = 0, row0 = 0, base = 0;
        if (s < a.sequences) {   // (the three loads together: one after the other they were a third of a small call)
            const int begin = a.cu_rows[s], end = a.cu_rows[s + 1], length = a.lengths[s];
            row0 = max(begin, 0);
            const int all = min(end, a.rows) - row0;
            n = min(all, a.max_rows);
            base = min(max(length, 0), a.pages_per_sequence * kQ4Page) - all;   // `n` is cut at max_rows
        }
        const int mine = n > 0 && (long long)n * group > a.tile_above ? (n * group + 2 * kRows - 1) / (2 * kRows) : 0;
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += other;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, before > place);
        if (found != 0) {
            const int at = __ffs(found) - 1;
            w.s = s0 + at;
            w.row0 = __shfl_sync(0xffffffffu, row0, at);
            w.n = __shfl_sync(0xffffffffu, n, at);
            const int pairs = __shfl_sync(0xffffffffu, mine, at), first = __shfl_sync(0xffffffffu, before, at) - pairs;
            w.flat0 = (pairs - 1 - (place - first)) * 2 * kRows;
            w.base = __shfl_sync(0xffffffffu, base, at);
            return true;
        }
        place -= __shfl_sync(0xffffffffu, before, 31);
    }
    return false;
}

template <int HD, bool PAIR>
__global__ void __launch_bounds__(Tile<HD, PAIR>::THREADS, 1) kvq4_tile_kernel(const KvQ4Attention a) {
    using T = Tile<HD, PAIR>;
    constexpr int NG = HD / 32, WORDS = NG, BLOCK = kQ4Page * 16 * WORDS, RECORD = q4_record(HD);
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int group = a.q_heads / a.kv_heads, kvh = (int)blockIdx.x % a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Work w;
    const int split = (int)blockIdx.x / a.kv_heads % a.tile_splits;
    if (!find_work(a, (int)blockIdx.x / a.kv_heads / a.tile_splits, lane, w)) return;
    const uint32_t at = smem_u32(smem), bars = at + T::BARS;
    const uint32_t q_full = bars, s_full = bars + 16, p_full = bars + 32, o_full = bars + 48, k_full = bars + 64, k_empty = bars + 80, v_full = bars + 96, v_empty = bars + 112,
                   drained = bars + 128, tmem_slot = bars + 144, failed = bars + 148;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 4 * T::HALVES); mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4 * T::HALVES); mbar_init(o_full + 8 * i, 1);
            mbar_init(k_full + 8 * i, kKWarps); mbar_init(k_empty + 8 * i, 1); mbar_init(v_full + 8 * i, kVWarps); mbar_init(v_empty + 8 * i, 1);
            mbar_init(drained + 8 * i, 1);
        }
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(failed), "r"(0) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == T::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);

    // a tile's rows and key tiles; key tiles begin at multiples of 128, the first one where the pair's first row looks
    int live[2], n[2];
    const int low = a.window > 0 ? max(0, w.base + w.flat0 / group - a.window + 1) : 0;
    int first_tile = low / kKeys;
    int high = 0;
    for (int t = 0; t < 2; ++t) {
        const int flat = w.flat0 + t * kRows;
        live[t] = max(0, min(kRows, w.n * group - flat));
        const int to = live[t] > 0 ? w.base + (flat + live[t] - 1) / group + 1 : 0;
        n[t] = max(0, (to + kKeys - 1) / kKeys - first_tile);
        if (to <= 0) n[t] = 0;
        high = max(high, to);
    }
    {   // this CTA's share of them
        const int share = (max(n[0], n[1]) + a.tile_splits - 1) / a.tile_splits, begin = split * share;
        first_tile += begin;
        n[0] = max(0, min(n[0] - begin, share));
        n[1] = max(0, min(n[1] - begin, share));
    }
    const int n_tiles = max(n[0], n[1]);
    // the sequence's keys as operands in memory, where the call has room for them
    const Tiles tiles = a.scratch_tiles > 0 ? tiles_before(a, w.s, lane) : Tiles{};
    const bool expanded = a.scratch_tiles > 0 && tiles.first + tiles.count <= a.scratch_tiles;
    const unsigned char* operands = a.scratch + ((long long)(tiles.first + first_tile - tiles.tile0) * a.kv_heads + kvh) * (T::K_TILE + T::V_TILE);
    const int32_t* table = a.page_tables + w.s * a.table_stride;
    const int table_pages = (high + kQ4Page - 1) / kQ4Page;   // those that some row looks at
    // A wait that runs out says so to the whole CTA, whose rows become NaN: barriers may then be a phase apart, so that its others' are not to be trusted
    bool alive = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (alive) {
            alive = mbar_wait(bar, parity & 1u, nullptr, 0, a.wait_polls);
            if (!alive) asm volatile("st.shared.u32 [%0], %1;" ::"r"(failed), "r"(1) : "memory");
        }
    };

    if (warp >= T::K_WARP) {
        if constexpr (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == T::MMA_WARP) {
            // ---------------- products (the warp as a whole, one elected lane in it) ----------------
            // (trip counts that the compiler knows to be the warp's keep addresses and descriptors in uniform registers)
            const int n0 = __shfl_sync(0xffffffffu, n[0], 0), n1 = __shfl_sync(0xffffffffu, n[1], 0), n_all = max(n0, n1);
            const bool leader = elect_one();
            const uint32_t q_desc = umma_desc(at, T::Q_STRIDE), k_desc = umma_desc(at + T::K_AT, T::K_STRIDE), v_desc = umma_desc(at + T::V_AT, T::V_STRIDE);
            auto scores = [&](int t, int j) {
                const uint32_t b = k_desc + (j % T::K_SLOTS) * (T::K_TILE >> 4), hi = q_desc + T::PLANES * t * (T::Q_TILE >> 4);
                if (leader && alive) {
                    if (PAIR) {
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) {
                            umma_ss(tmem + 128 * t, hi + (T::Q_TILE >> 4) + i * (2 * T::Q_STRIDE >> 4), b + i * (2 * T::K_STRIDE >> 4), umma_idesc(kKeys), (uint32_t)(i != 0));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        umma_ss(tmem + 128 * t, hi + i * (2 * T::Q_STRIDE >> 4), b + i * (2 * T::K_STRIDE >> 4), umma_idesc(kKeys), (uint32_t)(PAIR || i != 0));
                    }
                }
                if (leader) umma_commit(s_full + 8 * t);
            };
            auto values = [&](int t, int j, int count) {
                wait(p_full + 8 * t, j);
                tc_fence_after();
                const uint32_t goes_on = PAIR ? j % kWindow != 0 : j != 0, p_at = tmem + 128 * t, o_at = tmem + 256 + 128 * t, b = v_desc + (j % T::V_SLOTS) * (T::V_TILE >> 4);
                if (leader && alive) {
                    if (PAIR) {
#pragma unroll
                        for (int i = 0; i < kKeys / 16; ++i) {
                            umma_ts(o_at, p_at + 32 * (i >> 1) + 8 * (i & 1) + 16, b + i * (2 * T::V_STRIDE >> 4), umma_idesc(HD), goes_on | (uint32_t)(i != 0));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kKeys / 16; ++i) {
                        umma_ts(o_at, p_at + 32 * (i >> 1) + 8 * (i & 1), b + i * (2 * T::V_STRIDE >> 4), umma_idesc(HD), PAIR ? 1u : goes_on | (uint32_t)(i != 0));
                    }
                }
                if (leader && j + 1 == count) umma_commit(o_full + 8 * t);
            };
            // (a slot that nobody asks for again is not given back; nor is one after an expired wait, so that no loader fills a slot whose last
            // filling may not be complete)
            auto release_k = [&](int j) { if (leader && alive && j + T::K_SLOTS < n_all) umma_commit(k_empty + 8 * (j % T::K_SLOTS)); };
            auto release_v = [&](int j) { if (leader && alive && j + T::V_SLOTS < n_all) umma_commit(v_empty + 8 * (j % T::V_SLOTS)); };
            // (a barrier costs a hundred clocks and more even where it is complete: K and V are waited for once a step, while the
            // probabilities are on their way anyhow)
            auto wait_k = [&](int j) { wait(k_full + 8 * (j % T::K_SLOTS), j / T::K_SLOTS); };
            if (n_all > 0) wait_k(0);
            if (n0 > 0) { wait(q_full, 0); tc_fence_after(); scores(0, 0); }
            if (n1 > 0) { wait(q_full + 8, 0); tc_fence_after(); scores(1, 0); }
            if (n_all > 0) release_k(0);
#pragma unroll 1
            for (int j = 0; j < n_all; ++j) {
                wait(v_full + 8 * (j % T::V_SLOTS), j / T::V_SLOTS);
                if (j + 1 < n_all) wait_k(j + 1);
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    const int nt = t == 0 ? n0 : n1;
                    if (j < nt) values(t, j, nt);
                    if (t == 1) release_v(j);
                    if (j + 1 < nt) scores(t, j + 1);   // over the probabilities that the products above have read
                    if (t == 1 && j + 1 < n_all) release_k(j + 1);
                }
            }
            // what was issued comes to its end before the block, and its tensor memory, can (the rows' threads may have given up)
            if (leader) umma_commit(drained);
            mbar_wait(drained, 0, nullptr, 0, kQ4WaitPolls);
        } else {
            // ---------------- page records to operands ----------------
            const unsigned char* head = a.cache + (long long)kvh * RECORD;
            const long long page_stride = (long long)a.kv_heads * RECORD;
            // the number of page `lane & 7` of key tile j, -1 where no row looks
            auto look_up = [&](int j) -> int {
                const int p = (first_tile + j) * kTilePages + (lane & 7);
                return j < n_tiles && p < table_pages ? table[p] : -1;
            };
            auto landed = [&](uint32_t bar) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            const __half2 minus72 = __float2half2_rn(-72.0f);
            const bool is_k = warp < T::K_WARP + kKWarps;
            if (expanded) {   // a warp's share of each tile by one bulk copy
                const int part = is_k ? warp - T::K_WARP : warp - T::V_WARP, bytes = is_k ? T::K_TILE / kKWarps : part < 2 ? T::V_TILE / 8 * 3 : T::V_TILE / 4, slots = is_k ? T::K_SLOTS : T::V_SLOTS;
                const uint32_t full = is_k ? k_full : v_full, empty = is_k ? k_empty : v_empty, skip = is_k ? part * bytes : part * (T::V_TILE / 8 * 3), to = at + (is_k ? T::K_AT : T::V_AT) + skip;
                const unsigned char* from = operands + (is_k ? 0 : T::K_TILE) + skip;
                const long long step = (long long)a.kv_heads * (T::K_TILE + T::V_TILE);
                int j = 0;
                for (; j < n_tiles; ++j) {
                    const int slot = j % slots;
                    if (j >= slots) wait(empty + 8 * slot, j / slots - 1);
                    if (__any_sync(0xffffffffu, !alive)) break;
                    if (lane == 0) {
                        mbar_expect_tx(full + 8 * slot, bytes);
                        bulk_g2s(to + slot * (is_k ? T::K_TILE : T::V_TILE), from + j * step, bytes, full + 8 * slot);
                    }
                    __syncwarp();
                }
                // the copies land before the block can end, whoever still waits for them (a phase that another loader has left incomplete is waited
                // for to the limit)
                for (int i = max(0, j - slots); i < j; ++i) mbar_wait(full + 8 * (i % slots), (uint32_t)(i / slots) & 1u, nullptr, 0, kLandPolls);
            } else if (is_k) {
                int ids = look_up(0), next_ids = look_up(1);
                // lane = (quarter t, row i of eight): eight lanes store 128 bytes side by side
                const int kw = warp - T::K_WARP, t = lane >> 3, place = lane & 7, key[2] = {key_of_place(place), key_of_place(8 + place)};
                uint32_t code[2][WORDS], scale[2][NG / 2];
                auto fetch = [&](int page, int from) {
                    const int id = __shfl_sync(0xffffffffu, from, page);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int u = 0; u < NG / 2; ++u) scale[h][u] = 0u;
                        if (id >= 0 && id < a.pages) {
                            const unsigned char* p = head + id * page_stride;
                            load_words<WORDS>(p + (key[h] * 4 + t) * (4 * WORDS), code[h]);
                            load_words<NG / 2>(p + 16 * HD + key[h] * (2 * NG), scale[h]);
                        }
                    }
                };
                fetch(kw, ids);
#pragma unroll 1
                for (int j = 0; j < n_tiles; ++j) {
                    if (j >= T::K_SLOTS) wait(k_empty + 8 * (j % T::K_SLOTS), j / T::K_SLOTS - 1);
                    if (__any_sync(0xffffffffu, !alive)) break;
                    const uint32_t to = at + T::K_AT + (j % T::K_SLOTS) * T::K_TILE + t * T::K_STRIDE + place * 16;
#pragma unroll 1
                    for (int page = kw; page < kTilePages; page += kKWarps) {
                        uint32_t c[2][WORDS], sc[2][NG / 2];   // the next page's come under this one's arithmetic
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int u = 0; u < WORDS; ++u) c[h][u] = code[h][u];
#pragma unroll
                            for (int u = 0; u < NG / 2; ++u) sc[h][u] = scale[h][u];
                        }
                        const bool more = page + kKWarps < kTilePages;
                        fetch(more ? page + kKWarps : kw, more ? ids : next_ids);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int G = 0; G < NG; ++G) {
                                const __half2 s = as_half2(__byte_perm(sc[h][G >> 1], 0u, (G & 1) ? 0x3232u : 0x1010u));
                                uint32_t y[4];
                                word_values(c[h][G], s, __hmul2(s, minus72), y);
                                sts128(to + 4 * G * T::K_STRIDE + (page * kQ4Page + 8 * h) * 16, make_uint4(y[0], y[1], y[2], y[3]));
                            }
                        }
                    }
                    landed(k_full + 8 * (j % T::K_SLOTS));
                    ids = next_ids;
                    next_ids = look_up(j + 2);
                }
            } else {
                int ids = look_up(0), next_ids = look_up(1);
                // lane = (t / 2, dimension g of eight, t % 2): sixteen lanes store 128 bytes side by side
                const int vw = warp - T::V_WARP, g = (lane >> 1) & 7, t = (lane >> 4) * 2 + (lane & 1);
                uint32_t code[2][WORDS], scale[2][NG];
                auto fetch = [&](int page, int from) {
                    const int id = __shfl_sync(0xffffffffu, from, page);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int u = 0; u < NG; ++u) scale[h][u] = 0u;
                        if (id >= 0 && id < a.pages) {
                            const unsigned char* p = head + id * page_stride;
                            load_words<WORDS>(p + 8 * HD + h * (BLOCK / 2) + (g * 4 + t) * (4 * WORDS), code[h]);
                            load_words<NG>(p + 17 * HD + (4 * h + t) * (4 * NG), scale[h]);
                        }
                    }
                };
                fetch(vw, ids);
#pragma unroll 1
                for (int j = 0; j < n_tiles; ++j) {
                    if (j >= T::V_SLOTS) wait(v_empty + 8 * (j % T::V_SLOTS), j / T::V_SLOTS - 1);
                    if (__any_sync(0xffffffffu, !alive)) break;
                    const int key0 = (first_tile + j) * kKeys;
                    const bool edge = key0 < low || key0 + kKeys > high;   // what lies where no row looks may be anything
                    const uint32_t to = at + T::V_AT + (j % T::V_SLOTS) * T::V_TILE + (t >> 1) * T::V_STRIDE + g * 16 + (t & 1) * 8;
#pragma unroll 1
                    for (int page = vw; page < kTilePages; page += kVWarps) {
                        uint32_t c[2][WORDS], sc[2][NG];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int u = 0; u < WORDS; ++u) { c[h][u] = code[h][u]; sc[h][u] = scale[h][u]; }
                        }
                        const bool more = page + kVWarps < kTilePages;
                        fetch(more ? page + kVWarps : vw, more ? ids : next_ids);
                        if (edge) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int k = key0 + page * kQ4Page + 8 * h + 2 * t;
                                const uint32_t keep = (k >= low && k < high ? 0xffffu : 0u) | (k + 1 >= low && k + 1 < high ? 0xffff0000u : 0u);
#pragma unroll
                                for (int G = 0; G < NG; ++G) sc[h][G] &= keep;
                            }
                        }
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            uint32_t y0[4], y1[4];
                            const __half2 s0 = as_half2(sc[0][G]), s1 = as_half2(sc[1][G]);
                            word_values(c[0][G], s0, __hmul2(s0, minus72), y0);
                            word_values(c[1][G], s1, __hmul2(s1, minus72), y1);
#pragma unroll
                            for (int u = 0; u < 4; ++u) sts64(to + 2 * page * T::V_STRIDE + (32 * G + 8 * u) * 16, y0[u], y1[u]);
                        }
                    }
                    landed(v_full + 8 * (j % T::V_SLOTS));
                    ids = next_ids;
                    next_ids = look_up(j + 2);
                }
            }
        }
    } else {
        // ---------------- softmax: one row per thread ----------------
        if constexpr (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        constexpr int HALVES = T::HALVES, DH = HD / HALVES;   // dimensions of the result that a thread has
        const int t = warp / (4 * HALVES), part = (warp >> 2) % HALVES, row0 = (warp & 3) * 32, row = row0 + lane, flat0 = w.flat0 + t * kRows;
        const uint32_t q_tile = at + T::PLANES * t * T::Q_TILE;
        // the two warps of a row block (not PAIR): a barrier of their own, which can also tell whether any of their threads says so
        const int pair_barrier = 1 + 4 * t + (warp & 3);
        auto pair_sync = [&]() { asm volatile("barrier.cta.sync.aligned %0, 64;" ::"r"(pair_barrier) : "memory"); };
        auto pair_any = [&](bool mine) -> bool {
            uint32_t r;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(r) : "r"((uint32_t)mine), "r"(pair_barrier) : "memory");
            return r != 0;
        };
        const uint32_t factors = at + T::FACTORS + t * kRows * 4, mine_at = at + T::XCH + ((t * 2 + part) * kRows + row) * 4, other_at = at + T::XCH + ((t * 2 + 1 - part) * kRows + row) * 4;
        float factor = 0.0f;   // of this thread's row's scores
        const int own = t == 0 ? n[0] : n[1], live_rows = t == 0 ? live[0] : live[1];
        if (own > 0) {
            // the warp's 32 query rows: lane = (row of eight, 8-dimension piece of four), scaled so that a row's largest lies in [2^13, 2^14)
            const int sub = lane & 7, pc = lane >> 3;
            constexpr int PP = HD / 32, GROUPS = 4 / HALVES, WORDS8 = PAIR ? 8 : 4;   // pieces per lane and row; groups of eight rows
            uint32_t next[PP][WORDS8];   // (a loop, the next group's loads under this one's arithmetic: straight code is fetched as slowly as data)
            auto ask = [&](int rg) {
                const int r = row0 + rg * 8 + sub;
                const long long from = (w.row0 + (flat0 + r) / group) * a.q_stride + (long long)(kvh * group + (flat0 + r) % group) * HD + pc * 8;
#pragma unroll
                for (int p = 0; p < PP; ++p) {
#pragma unroll
                    for (int u = 0; u < WORDS8; ++u) next[p][u] = 0u;
                    if (r < live_rows) q4_load_raw(a.q, from + p * 32, a.vector_q, next[p]);
                }
            };
            ask(GROUPS * part);
#pragma unroll 1
            for (int rg = GROUPS * part; rg < GROUPS * (part + 1); ++rg) {
                const int r = row0 + rg * 8 + sub;
                float x[PP][8];
                uint32_t top = 0;   // the largest magnitude's bits, which order as the values do, NaN above all
#pragma unroll
                for (int p = 0; p < PP; ++p) {
                    q4_values(next[p], a.type, x[p]);
#pragma unroll
                    for (int u = 0; u < 8; ++u) top = max(top, __float_as_uint(x[p][u]) & 0x7fffffffu);
                }
                if (rg + 1 < GROUPS * (part + 1)) ask(rg + 1);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
                // A row that is not finite is NaN where it sees a key.  Its operand is zero, so that its thread can tell, by the reference, whether it does;
                // its factor's sign tells the thread.
                const bool spoiled = top >= 0x7f800000u;
                const uint32_t keep = spoiled ? 0u : 0xffffffffu;
                const int e = top > 0 && !spoiled ? max(-126, min(126, 140 - (int)(top >> 23))) : 0;
                const float up = __int_as_float((e + 127) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f), f = __int_as_float((127 - e) << 23);
                const float size = q4_factor(f * fabsf(a.scale)), scaled = spoiled ? -size : size;
                if constexpr (HALVES == 1) {
                    const float of_row = __shfl_sync(0xffffffffu, scaled, lane & 7);
                    if ((lane >> 3) == rg) factor = of_row;
                } else if (pc == 0) {
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(factors + r * 4), "f"(scaled) : "memory");
                }
#pragma unroll
                for (int p = 0; p < PP; ++p) {
                    uint4 hi, lo;
                    uint32_t *h = &hi.x, *l = &lo.x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (PAIR) split2(x[p][i] * up, x[p][i + 4] * up, h[i], l[i]);
                        else h[i] = as_bits(__floats2half2_rn(x[p][i] * up, x[p][i + 4] * up));
                        h[i] &= keep;
                        if (PAIR) l[i] &= keep;
                    }
                    const uint32_t to = q_tile + (p * 4 + pc) * T::Q_STRIDE + r * 16;
                    sts128(to, hi);
                    if (PAIR) sts128(to + T::Q_TILE, lo);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * t);
            if constexpr (HALVES == 2) {
                pair_sync();
                factor = __uint_as_float(lds32(factors + row * 4));
            }
        }
        const bool spoiled = factor < 0.0f;
        factor = fabsf(factor);
        const bool have = row < live_rows;
        const int limit = have ? w.base + (flat0 + row) / group : -1, lowest = a.window > 0 ? limit - a.window + 1 : 0;
        // keys that every row of the warp sees
        const int all_high = __reduce_min_sync(0xffffffffu, limit), all_low = __reduce_max_sync(0xffffffffu, lowest);
        const uint32_t lanes = (uint32_t)row0 << 16, s_at = tmem + lanes + 128 * t, o_at = s_at + 256;
        float m = PAIR ? -INFINITY : kUnset;   // the reference: a score, or (not PAIR) an integer in base 2
        float2 l = make_float2(0.0f, 0.0f);   // the row's sum in two parts
        float sum[PAIR ? HD : 1], since = 1.0f;   // earlier windows' results; the factor that has come to them since the last one's end
#pragma unroll
        for (int i = 0; i < (PAIR ? HD : 1); ++i) sum[i] = 0.0f;
        // the number of page `lane & 7` of a tile, compared a step later, so that nothing waits for it
        const int32_t* ahead = table + first_tile * kTilePages + (lane & 7);
        int left = table_pages - first_tile * kTilePages - (lane & 7);
        auto look_up = [&]() -> int {
            const int id = left > 0 ? *ahead : 0;
            ahead += kTilePages;
            left -= kTilePages;
            return id;
        };
        int next_id = own > 0 ? look_up() : 0;
        for (int j = 0; j < own; ++j) {
            const uint32_t bad = __ballot_sync(0xffffffffu, next_id < 0 || next_id >= a.pages) & 0xffu;   // pages outside of the arena
            next_id = look_up();
            wait(s_full + 8 * t, j);
            tc_fence_after();
            const int key0 = (first_tile + j) * kKeys;
            const bool masked = key0 + kKeys - 1 > all_high || key0 < all_low || bad != 0;
            const bool fresh = PAIR ? j % kWindow == 0 : j == 0;
            if (PAIR && fresh && j > 0) {   // (the scores' barrier also says that the products into O so far are complete)
#pragma unroll
                for (int i = 0; i < HD; i += 32) {
                    float o[32];
                    tmem_ld32(o_at + i, o);
                    tmem_wait_ld();
                    tmem_tie32(o);
#pragma unroll
                    for (int u = 0; u < 32; ++u) sum[PAIR ? i + u : 0] = fmaf(sum[PAIR ? i + u : 0], since, o[u]);
                }
                since = 1.0f;
            }
            auto hide = [&](float (&s)[32], int i) {
#pragma unroll
                for (int u = 0; u < 32; ++u) {
                    const int key = key0 + i + (u & 16) + key_of_place(u & 15);
                    if (key > limit || key < lowest || ((bad >> ((i + u) >> 4)) & 1u)) s[u] = -INFINITY;
                }
            };
            // What has been summed, as the row's reference moves: times f
            auto rescale = [&](float f) {
                l.x *= f; l.y *= f;
                if (PAIR) since *= f;
                if (fresh) return;
#pragma unroll 1
                for (int i = part * DH; i < (part + 1) * DH; i += 16) {
                    float o[2][8];
                    tmem_ld8(o_at + i, o[0]);
                    tmem_ld8(o_at + i + 8, o[1]);
                    tmem_wait_ld();
                    tmem_tie(o[0]);
                    tmem_tie(o[1]);
                    uint32_t r[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) r[u] = __float_as_uint(o[u >> 3][u & 7] * f);
                    tmem_st16(o_at + i, r);
                }
            };
            if constexpr (PAIR) {   // the rows' sums take the registers: scores 32 at a time, twice
                float s[32], mx = -INFINITY;
#pragma unroll 1
                for (int i = 0; i < kKeys; i += 32) {
                    tmem_ld32(s_at + i, s);
                    tmem_wait_ld();
                    tmem_tie32(s);
                    if (masked) hide(s, i);
                    mx = fmaxf(mx, most_of(s));
                }
                const bool moves = mx > m && (m == -INFINITY || (mx - m) * factor > kSlack);
                if (__any_sync(0xffffffffu, moves)) {
                    const float f = moves ? (m == -INFINITY ? 0.0f : exp2_approx((m - mx) * factor)) : 1.0f;
                    if (moves) m = mx;
                    rescale(f);
                }
                const float shift = m == -INFINITY ? 0.0f : kHeld - __fmul_rn(m, factor);
                float2 tile = make_float2(0.0f, 0.0f);
#pragma unroll 1
                for (int i = 0; i < kKeys; i += 32) {
                    tmem_ld32(s_at + i, s);
                    tmem_wait_ld();
                    tmem_tie32(s);
                    if (masked) hide(s, i);
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        // (rounded before the reference is taken off, as the reference is: the largest score's difference is zero however large)
                        const float2 y = __fadd2_rn(make_float2(__fmul_rn(s[2 * u], factor), __fmul_rn(s[2 * u + 1], factor)), make_float2(shift, shift));
                        const float2 p = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        tile = __fadd2_rn(tile, p);
                        split2(p.x, p.y, hi[u], lo[u]);
                    }
                    tmem_st16(s_at + i, hi);   // over the 32 scores just read
                    tmem_st16(s_at + i + 16, lo);
                }
                // A tile's sum joins the row's with what the addition rounds off kept beside it (Knuth's two-sum): one by one, thousands of keys of
                // 2^-25 of the largest were lost (1,120 rows, 11,557 keys, heads of 64: all values 5.1e-6 off 64 bits, rows with one key of 0.99
                // 3e-5; so 7.0e-7, the plain form 1.9e-6)
                const float add = tile.x + tile.y, to = l.x + add, rest = to - l.x;
                l.y += (l.x - (to - rest)) + (add - rest);
                l.x = to;
            } else {
                if (j == 0) {   // the first reference, from the first scores
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int i = 64 * part; i < 64 * part + 64; i += 32) {
                        float s[32];
                        tmem_ld32(s_at + i, s);
                        tmem_wait_ld();
                        tmem_tie32(s);
                        if (masked) hide(s, i);
                        mx = fmaxf(mx, most_of(s));
                    }
                    mx *= factor;
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine_at), "f"(mx) : "memory");
                    pair_sync();
                    mx = fmaxf(mx, __uint_as_float(lds32(other_at)));
                    if (mx > kUnset) m = ceilf(mx);   // (not where no key is seen yet, and not for NaN)
                    pair_sync();   // (the words are written again where a score passes the reference)
                }
                // Probabilities of 32 scores at a time against the reference as it is, their maximum found beside them.  Where a score of the
                // row passes the reference by more than the slack (a row's first keys, hardly ever later) the reference, an integer,
                // moves up in both of the row's threads, what has been summed and this tile's earlier probabilities are divided by the power of
                // two, and the 32 are done again: the scores still lie there.
#pragma unroll 1
                for (int i = 64 * part; i < 64 * part + 64; i += 32) {
                    uint32_t hi[16];
                    float l0, l1;
                    for (;;) {
                        float s[32], mx;
                        tmem_ld32(s_at + i, s);
                        const float shift = kHeld - m;
                        l0 = l1 = 0.0f;
                        // so large that a fused multiply-add's exact product is far from the reference, a rounded one: round first
                        const bool large = __any_sync(0xffffffffu, fabsf(m) > 4194304.0f && m != kUnset);
                        const float times = large ? 1.0f : factor;
                        tmem_wait_ld();
                        tmem_tie32(s);
                        if (masked) hide(s, i);
                        if (large) {
#pragma unroll
                            for (int u = 0; u < 32; ++u) s[u] *= factor;
                        }
                        mx = most_of(s) * times;
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const float2 y = __ffma2_rn(make_float2(s[2 * u], s[2 * u + 1]), make_float2(times, times), make_float2(shift, shift));
                            const float2 p = (u * kPolynomial) % 16 < kPolynomial ? exp2_pair(y) : make_float2(exp2_approx(y.x), exp2_approx(y.y));
                            const __half2 rounded = __floats2half2_rn(p.x, p.y);   // what the products take
                            const float2 lp = __fadd2_rn(make_float2(l0, l1), __half22float2(rounded));
                            l0 = lp.x;
                            l1 = lp.y;
                            hi[u] = as_bits(rounded);
                        }
                        if (!pair_any(mx > m + kSlack)) break;
                        tmem_wait_st();   // what is read back below may have been stored in this tile: earlier probabilities, sums of an earlier move
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine_at), "f"(mx) : "memory");
                        pair_sync();
                        mx = fmaxf(mx, __uint_as_float(lds32(other_at)));
                        const bool moves = mx > m + kSlack;
                        const float to = moves ? ceilf(mx) : m;
                        const float f = moves ? (m - to < -126.0f ? 0.0f : power2((int)(m - to))) : 1.0f;
                        m = to;
                        rescale(f);
                        const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
                        for (int e = 64 * part; e < i; e += 16) {
                            const uint32_t place = s_at + (e & ~31) + (e & 16) / 2;
                            float p[8];
                            tmem_ld8(place, p);
                            tmem_wait_ld();
                            tmem_tie(p);
                            uint32_t r[8];
#pragma unroll
                            for (int u = 0; u < 8; ++u) r[u] = as_bits(__hmul2(as_half2(__float_as_uint(p[u])), f2));
                            tmem_st8(place, r);
                        }
                    }
                    l.x += l0;
                    l.y += l1;
                    tmem_st16(s_at + i, hi);   // over these scores
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * t);
        }
        if (own > 0) {
            wait(o_full + 8 * t, 0);
            tc_fence_after();
        }
        // rows to memory through the shared memory that the queries have left: a warp's own rows, in 16-byte pieces by number ^ (row % 8)
        if (live_rows > row0) {
            constexpr int VALUE = PAIR ? 4 : 2, ROW_BYTES = DH * VALUE, PIECES = ROW_BYTES / 16, SWAP = PIECES < 8 ? PIECES - 1 : 7;
            float total = l.x + l.y;
            const bool none = own == 0 || m == (PAIR ? -INFINITY : kUnset);   // no key seen
            if (spoiled && !none) total = __int_as_float(0x7fffffff);
            if constexpr (HALVES == 2) {
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine_at), "f"(total) : "memory");
                pair_sync();
                const float other = __uint_as_float(lds32(other_at));
                total = part == 0 ? total + other : other + total;
            }
            // where the keys are shared with other CTAs: the row's sums, for the merge
            const bool shared = a.tile_splits > 1, have_row = row < live_rows;
            float* record = a.tile_partial + (((long long)(w.row0 + (flat0 + row) / group) * a.q_heads + kvh * group + (flat0 + row) % group) * a.tile_splits + split) * (HD + 4);
            if (shared && have_row && part == 0) {
                record[HD] = !alive || lds32(failed) != 0 || total != total ? __int_as_float(0x7fffffff) : none ? -INFINITY : PAIR ? __fmul_rn(m, factor) : m;
                record[HD + 1] = total;
            }
            const uint32_t stage = q_tile + ((warp & 3) * HALVES + part) * 32 * ROW_BYTES;
            float inv = total > 0.0f ? 1.0f / total : total != total ? total : 0.0f;
            if (!alive || lds32(failed) != 0) inv = __int_as_float(0x7fffffff);
            if (own > 0) {
#pragma unroll
                for (int i = 0; i < DH; i += 32) {
                    float o[32];
                    tmem_ld32(o_at + part * DH + i, o);
                    tmem_wait_ld();
                    tmem_tie32(o);
#pragma unroll
                    for (int u = 0; u < 32; ++u) {
                        if (PAIR) o[u] = fmaf(sum[PAIR ? i + u : 0], since, o[u]);
                        if (!shared) o[u] = inv != 0.0f ? o[u] * inv : 0.0f;
                    }
                    if (shared) {
#pragma unroll
                        for (int u = 0; u < 32; u += 4) {
                            if (have_row) *reinterpret_cast<float4*>(record + part * DH + i + u) = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
                        }
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 32; u += 16 / VALUE) {
                        uint4 v;
                        if (PAIR) {
                            v = make_uint4(__float_as_uint(o[u]), __float_as_uint(o[u + 1]), __float_as_uint(o[u + 2]), __float_as_uint(o[u + 3]));
                        } else {
                            uint32_t* p = &v.x;
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                if (a.type == kQ4F16) p[x] = as_bits(__floats2half2_rn(o[(u + 2 * x) & 31], o[(u + 2 * x + 1) & 31]));
                                else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[x]) : "f"(o[(u + 2 * x + 1) & 31]), "f"(o[(u + 2 * x) & 31]));
                            }
                        }
                        sts128(stage + lane * ROW_BYTES + ((((i + u) * VALUE / 16) ^ (lane & SWAP)) << 4), v);
                    }
                }
            } else {   // no key for any row of the tile
#pragma unroll
                for (int i = 0; i < PIECES; ++i) sts128(stage + lane * ROW_BYTES + (i << 4), make_uint4(0u, 0u, 0u, 0u));
            }
            __syncwarp();
            constexpr int PER = 32 / PIECES;   // rows per pass
#pragma unroll 1
            for (int r0 = 0; r0 < 32 && !shared; r0 += PER) {
                const int r = r0 + lane / PIECES, p = lane % PIECES, flat = flat0 + row0 + r;
                if (row0 + r >= live_rows) continue;
                const uint4 v = lds128(stage + r * ROW_BYTES + ((p ^ (r & SWAP)) << 4));
                const long long to = (w.row0 + flat / group) * a.out_stride + (long long)(kvh * group + flat % group) * HD + part * DH + p * (16 / VALUE);
                if (a.vector_out) {
                    *reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.out) + to * VALUE) = v;
                } else {
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (PAIR) {
                            static_cast<uint32_t*>(a.out)[to + i] = x[i];
                        } else {
                            static_cast<unsigned short*>(a.out)[to + 2 * i] = (unsigned short)x[i];
                            static_cast<unsigned short*>(a.out)[to + 2 * i + 1] = (unsigned short)(x[i] >> 16);
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == T::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// A row's sums over its key tiles' shares: out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), shares in order, a warp per (row, query head).
template <int HD>
__global__ void __launch_bounds__(128) kvq4_tile_merge_kernel(const KvQ4Attention a) {
    constexpr int PER = HD / 32;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, row = (int)(id / a.q_heads), qh = (int)(id % a.q_heads), group = a.q_heads / a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (row >= a.rows) return;
    int s = 0, above = a.sequences;   // the last sequence that begins at or before the row
    while (above - s > 1) {
        const int mid = (s + above) / 2;
        if (a.cu_rows[mid] <= row) s = mid; else above = mid;
    }
    const int row0 = max(a.cu_rows[s], 0), n = min(min(a.cu_rows[s + 1], a.rows) - row0, a.max_rows);
    if (row < row0 || row >= row0 + n || (long long)n * group <= a.tile_above) return;   // not the tile kernel's
    const float* from = a.tile_partial + id * a.tile_splits * (HD + 4);
    float top = -INFINITY;
    for (int i = lane; i < a.tile_splits; i += 32) top = fmaxf(top, __ldcg(from + (long long)i * (HD + 4) + HD));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum[PER], total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] = 0.0f;
    for (int i = 0; i < a.tile_splits; ++i) {
        const float* rec = from + (long long)i * (HD + 4);
        const float m = __ldcg(rec + HD);
        if (m == -INFINITY) continue;   // no key: its values were not written
        const float f = exp2_approx(m - top);
        total = fmaf(__ldcg(rec + HD + 1), f, total);
#pragma unroll
        for (int u = 0; u < PER; ++u) sum[u] = fmaf(__ldcg(rec + lane + 32 * u), f, sum[u]);
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const float x = total > 0.0f || total != total ? sum[u] / total : 0.0f;
        const long long to = row * a.out_stride + (long long)qh * HD + lane + 32 * u;
        if (a.type == kQ4F32) static_cast<float*>(a.out)[to] = x;
        else if (a.type == kQ4F16) static_cast<__half*>(a.out)[to] = __float2half_rn(x);
        else asm volatile("{\n\t.reg .b16 t;\n\tcvt.rn.bf16.f32 t, %1;\n\tst.global.b16 [%0], t;\n\t}" ::"l"(static_cast<unsigned short*>(a.out) + to), "f"(x) : "memory");
    }
}

// Page records as the operands above: a CTA has one key tile of one kv head, a warp one of its eight pages.
template <int HD>
__global__ void __launch_bounds__(kTilePages * 32) kvq4_expand_kernel(const KvQ4Attention a) {
    using T = Tile<HD, false>;
    constexpr int NG = HD / 32, WORDS = NG, BLOCK = kQ4Page * 16 * WORDS, RECORD = q4_record(HD);
    const int page = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = (int)blockIdx.x % a.kv_heads, place = (int)blockIdx.x / a.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int s = -1, j = 0, low = 0, high = 0, tile0 = 0;
    int before = 0;
    for (int s0 = 0; s0 < a.sequences && s < 0; s0 += 32) {   // every warp by itself
        int t0 = 0, l = 0, h = 0;
        const int mine = s0 + lane < a.sequences ? tiles_of(a, s0 + lane, t0, l, h) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, before + upto > place);
        if (found != 0) {
            const int at = __ffs(found) - 1, end = before + __shfl_sync(0xffffffffu, upto, at), count = __shfl_sync(0xffffffffu, mine, at);
            if (end > a.scratch_tiles) return;   // the sequence's operands do not fit: its CTAs convert for themselves
            s = s0 + at;
            j = place - (end - count);
            tile0 = __shfl_sync(0xffffffffu, t0, at); low = __shfl_sync(0xffffffffu, l, at); high = __shfl_sync(0xffffffffu, h, at);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (s < 0) return;
    const int key0 = (tile0 + j) * kKeys + page * kQ4Page, index = key0 / kQ4Page;
    const int id = key0 < high ? a.page_tables[s * a.table_stride + index] : -1;
    const bool have = id >= 0 && id < a.pages;
    const unsigned char* p = a.cache + ((long long)(have ? id : 0) * a.kv_heads + kvh) * RECORD;
    unsigned char* out = a.scratch + ((long long)place * a.kv_heads + kvh) * (T::K_TILE + T::V_TILE);
    const __half2 minus72 = __float2half2_rn(-72.0f);
    {
        const int t = lane >> 3, r = lane & 7;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key = key_of_place(8 * h + r);
            uint32_t c[WORDS], sc[NG / 2];
#pragma unroll
            for (int u = 0; u < NG / 2; ++u) sc[u] = 0u;
#pragma unroll
            for (int u = 0; u < WORDS; ++u) c[u] = 0u;
            if (have) {
                load_words<WORDS>(p + (key * 4 + t) * (4 * WORDS), c);
                load_words<NG / 2>(p + 16 * HD + key * (2 * NG), sc);
            }
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                const __half2 scale = as_half2(__byte_perm(sc[G >> 1], 0u, (G & 1) ? 0x3232u : 0x1010u));
                uint32_t y[4];
                word_values(c[G], scale, __hmul2(scale, minus72), y);
                *reinterpret_cast<uint4*>(out + (4 * G + t) * T::K_STRIDE + (page * kQ4Page + 8 * h + r) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
            }
        }
    }
    {
        const int g = (lane >> 1) & 7, t = (lane >> 4) * 2 + (lane & 1);
        uint32_t c[2][WORDS], sc[2][NG];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int u = 0; u < WORDS; ++u) c[h][u] = sc[h][u] = 0u;
            if (have) {
                load_words<WORDS>(p + 8 * HD + h * (BLOCK / 2) + (g * 4 + t) * (4 * WORDS), c[h]);
                load_words<NG>(p + 17 * HD + (4 * h + t) * (4 * NG), sc[h]);
            }
            const int k = key0 + 8 * h + 2 * t;   // what lies where no row looks may be anything
            const uint32_t keep = (k >= low && k < high ? 0xffffu : 0u) | (k + 1 >= low && k + 1 < high ? 0xffff0000u : 0u);
#pragma unroll
            for (int G = 0; G < NG; ++G) sc[h][G] &= keep;
        }
#pragma unroll
        for (int G = 0; G < NG; ++G) {
            uint32_t y0[4], y1[4];
            const __half2 s0 = as_half2(sc[0][G]), s1 = as_half2(sc[1][G]);
            word_values(c[0][G], s0, __hmul2(s0, minus72), y0);
            word_values(c[1][G], s1, __hmul2(s1, minus72), y1);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                *reinterpret_cast<uint2*>(out + T::K_TILE + (2 * page + (t >> 1)) * T::V_STRIDE + (32 * G + 8 * u + g) * 16 + (t & 1) * 8) = make_uint2(y0[u], y1[u]);
            }
        }
    }
}

template <int HD, bool PAIR>
cudaError_t launch_tile(cudaStream_t stream, KvQ4Attention a) {
    static bool configured[kMaxDevices] = {false};   // function attributes are per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kvq4_tile_kernel<HD, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tile<HD, PAIR>::SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    // at most this many pairs of tiles, however the rows are spread over the sequences
    const long long places = kvq4_tile_places(a);
    if (places * a.tile_splits * a.kv_heads > 0x7fffffffll) return cudaErrorInvalidValue;
    if (places <= 0) return cudaSuccess;
    const auto launch = [&](auto kernel, long long grid, int threads, size_t smem) {   // early: see launch_rows
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3((unsigned)threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, a);
    };
    if (a.scratch_tiles > 0) {
        e = launch(kvq4_expand_kernel<HD>, (long long)a.scratch_tiles * a.kv_heads, kTilePages * 32, 0);
        if (e != cudaSuccess) return e;
    }
    e = launch(kvq4_tile_kernel<HD, PAIR>, places * a.tile_splits * a.kv_heads, Tile<HD, PAIR>::THREADS, Tile<HD, PAIR>::SMEM);
    if (e == cudaSuccess && a.tile_splits > 1) e = launch(kvq4_tile_merge_kernel<HD>, ((long long)a.rows * a.q_heads + 3) / 4, 128, 0);
    return e;
}

}  // namespace

long long kvq4_tile_places(const KvQ4Attention& a) {
    const long long flats = (long long)a.rows * (a.q_heads / a.kv_heads);
    return flats / (2 * kRows) + std::min<long long>(a.sequences, flats / (a.tile_above + 1));
}

cudaError_t launch_kvq4_tiles(cudaStream_t stream, const KvQ4Attention& a) {
    const bool pair = a.type == kQ4F32;
    if (a.head_dim == 64) return pair ? launch_tile<64, true>(stream, a) : launch_tile<64, false>(stream, a);
    if (a.head_dim == 128) return pair ? launch_tile<128, true>(stream, a) : launch_tile<128, false>(stream, a);
    return cudaErrorInvalidValue;
}

}  // namespace ribn
