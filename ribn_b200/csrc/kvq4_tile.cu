// Attention of many query rows per sequence over the 4-bit paged KV cache (kvq4.cuh) on the tcgen05 tensor cores.
//
// A CTA serves one (sequence, kv head) and two tiles of 128 query rows (row = row of the sequence x query head of the group), each
// with softmax warps of its own, so that one tile's products run while the other's probabilities are formed.  Per 128 keys:
//   S = Q K^T   A = the queries as binary16 in shared memory, scaled by a power of two per row, B = K;
//   P           a thread owns a row: softmax in base 2 against a reference that moves only when a score passes it by 2^8, P (held
//               2^7 times) as binary16 over S in tensor memory;
//   O += P V    A = P from tensor memory, B = V^T.
// Seven warps turn page records into those operands, registers to shared memory: a nibble under the exponent of 64 is 64 + code,
// one fused multiply-add with the scale and -72 x scale, both exact, gives the value.  Sums over dimensions and keys may run in any order,
// so neither operand is reordered: of K the word's pairs (i, i + 4) stay neighbours and the queries' dimensions follow, of V a lane's keys
// 2 t, 2 t + 1, 2 t + 8, 2 t + 9 stay neighbours and the rows of K follow.
// F32 queries and probabilities are binary16 hi + lo pairs, two products each; as an addition in tensor memory cuts at the sum's last
// bit, their sums over 256 keys move into the rows' registers.
// Roles of the 16 warps: 0..3 / 4..7 softmax and output of tile 0 / 1, 8..11 K, 12 issues the products, 13..15 V.  Every wait is
// bounded; where one runs out the CTA's rows become NaN.
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

#include "kvq4.cuh"
#include "tmem.cuh"

namespace ribn {

namespace {

constexpr int kRows = 128, kKeys = 128, kThreads = 512;
constexpr int kMmaWarp = 12, kKWarp0 = 8, kKWarps = 4, kVWarp0 = 13, kVWarps = 3;
constexpr int kTilePages = kKeys / kQ4Page;
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr float kLog2e = 1.4426950408889634f, kHeld = 7.0f, kSlack = 8.0f;
constexpr int kWindow = 2;   // PAIR: key tiles whose products one sum in tensor memory holds

template <int HD, bool PAIR>
struct Tile {
    static constexpr int PIECES = HD / 8;                         // 16-byte pieces of a query or key row
    static constexpr int Q_STRIDE = kRows * 16, Q_TILE = PIECES * Q_STRIDE;
    // 32 and 64 bytes of padding keep the four quarters of a lane group's stores in banks of their own
    static constexpr int K_STRIDE = kKeys * 16 + 32, K_TILE = PIECES * K_STRIDE;
    static constexpr int V_STRIDE = HD * 16 + 64, V_TILE = kKeys / 8 * V_STRIDE;
    static constexpr int PLANES = PAIR ? 2 : 1, K_SLOTS = 2, V_SLOTS = PAIR ? 1 : 2;
    static constexpr int K_AT = 2 * PLANES * Q_TILE, V_AT = K_AT + K_SLOTS * K_TILE, BARS = V_AT + V_SLOTS * V_TILE;
    static constexpr size_t SMEM = BARS + 192;
    // 512 x 128 registers at launch: softmax, the others
    static constexpr int SOFTMAX_REGS = PAIR ? 192 : 160, OTHER_REGS = PAIR ? 64 : 96;
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
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
// A column of a key tile holds key (column & ~15) + key_of_place(column & 15)
__device__ __forceinline__ constexpr int key_of_place(int p) { return 2 * (p >> 2) + (p & 1) + 8 * ((p >> 1) & 1); }

// The pair of query tiles of this CTA: sequences in order, each one's later rows, which have the most keys, first.
struct Work {
    int s, row0, n, base, flat0;   // flat0: first query row of tile 0
};
__device__ __forceinline__ bool find_work(const KvQ4Attention& a, int place, int lane, Work& w) {
    const int group = a.q_heads / a.kv_heads;
    for (int s0 = 0; s0 < a.sequences; s0 += 32) {
        const int s = s0 + lane;
        int n = 0, row0 = 0;
        if (s < a.sequences) {
            row0 = max(a.cu_rows[s], 0);
            n = min(min(a.cu_rows[s + 1], a.rows) - row0, a.max_rows);
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
            const int all = min(a.cu_rows[w.s + 1], a.rows) - w.row0;   // `n` is cut at max_rows
            w.base = min(max(a.lengths[w.s], 0), a.pages_per_sequence * kQ4Page) - all;
            return true;
        }
        place -= __shfl_sync(0xffffffffu, before, 31);
    }
    return false;
}

template <int HD, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) kvq4_tile_kernel(const KvQ4Attention a) {
    using T = Tile<HD, PAIR>;
    constexpr int NG = HD / 32, WORDS = NG, BLOCK = kQ4Page * 16 * WORDS, RECORD = q4_record(HD);
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int group = a.q_heads / a.kv_heads, kvh = (int)blockIdx.x % a.kv_heads;
    Work w;
    if (!find_work(a, (int)blockIdx.x / a.kv_heads, lane, w)) return;
    const uint32_t at = smem_u32(smem), bars = at + T::BARS;
    const uint32_t q_full = bars, s_full = bars + 16, p_full = bars + 32, o_full = bars + 48, k_full = bars + 64, k_empty = bars + 80, v_full = bars + 96, v_empty = bars + 112,
                   drained = bars + 128, tmem_slot = bars + 136, failed = bars + 140;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 4); mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, 4); mbar_init(o_full + 8 * i, 1);
            mbar_init(k_full + 8 * i, kKWarps); mbar_init(k_empty + 8 * i, 1); mbar_init(v_full + 8 * i, kVWarps); mbar_init(v_empty + 8 * i, 1);
        }
        mbar_init(drained, 1);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(failed), "r"(0) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);

    // a tile's rows and key tiles; key tiles begin at multiples of 128, the first one where the pair's first row looks
    int live[2], n[2];
    const int low = a.window > 0 ? max(0, w.base + w.flat0 / group - a.window + 1) : 0, first_tile = low / kKeys;
    int high = 0;
    for (int t = 0; t < 2; ++t) {
        const int flat = w.flat0 + t * kRows;
        live[t] = max(0, min(kRows, w.n * group - flat));
        const int to = live[t] > 0 ? w.base + (flat + live[t] - 1) / group + 1 : 0;
        n[t] = max(0, (to + kKeys - 1) / kKeys - first_tile);
        if (to <= 0) n[t] = 0;
        high = max(high, to);
    }
    const int n_tiles = max(n[0], n[1]);
    const int32_t* table = a.page_tables + w.s * a.table_stride;
    const int table_pages = (high + kQ4Page - 1) / kQ4Page;   // those that some row looks at
    bool alive = true;

    if (warp >= kKWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::OTHER_REGS));
        if (warp == kMmaWarp) {
            // ---------------- products (the warp as a whole, one elected lane in it) ----------------
            const bool leader = elect_one();
            const uint32_t q_desc = umma_desc(at, T::Q_STRIDE), k_desc = umma_desc(at + T::K_AT, T::K_STRIDE), v_desc = umma_desc(at + T::V_AT, T::V_STRIDE);
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (alive) {
                    alive = mbar_wait(bar, parity & 1u, nullptr, 0, kSpinLimit);
                    if (!alive && lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(failed), "r"(1) : "memory");
                }
            };
            auto scores = [&](int t, int j) {
                wait(k_full + 8 * (j % T::K_SLOTS), j / T::K_SLOTS);
                tc_fence_after();
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
            auto values = [&](int t, int j) {
                wait(p_full + 8 * t, j);
                wait(v_full + 8 * (j % T::V_SLOTS), j / T::V_SLOTS);
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
                if (leader && j + 1 == n[t]) umma_commit(o_full + 8 * t);
            };
            // (a slot that nobody asks for again is not given back: the arrival could come after the block's end)
            auto release_k = [&](int j) { if (leader && j + T::K_SLOTS < n_tiles) umma_commit(k_empty + 8 * (j % T::K_SLOTS)); };
            auto release_v = [&](int j) { if (leader && j + T::V_SLOTS < n_tiles) umma_commit(v_empty + 8 * (j % T::V_SLOTS)); };
            for (int t = 0; t < 2; ++t) {
                if (n[t] == 0) continue;
                wait(q_full + 8 * t, 0);
                scores(t, 0);
            }
            if (n_tiles > 0) release_k(0);
            for (int j = 0; j < n_tiles; ++j) {
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    if (j < n[t]) values(t, j);
                    if (t == 1) release_v(j);
                    if (j + 1 < n[t]) scores(t, j + 1);   // over the probabilities that the products above have read
                    if (t == 1 && j + 1 < n_tiles) release_k(j + 1);
                }
            }
            if (!alive) {
                // let what was issued come to its end before the block, and its tensor memory, can
                if (leader) umma_commit(drained);
                mbar_wait(drained, 0, nullptr, 0, kSpinLimit);
            }
        } else {
            // ---------------- page records to operands ----------------
            const int g = lane >> 2, t = lane & 3;
            const unsigned char* head = a.cache + (long long)kvh * RECORD;
            const long long page_stride = (long long)a.kv_heads * RECORD;
            // the number of page `lane & 7` of key tile j, -1 where no row looks or outside of the arena
            auto look_up = [&](int j) -> int {
                const int p = (first_tile + j) * kTilePages + (lane & 7);
                const int id = j < n_tiles && p < table_pages ? table[p] : -1;
                return id >= 0 && id < a.pages ? id : -1;
            };
            auto landed = [&](uint32_t bar) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (alive) {
                    alive = mbar_wait(bar, parity & 1u, nullptr, 0, kSpinLimit);
                    if (!alive && lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(failed), "r"(1) : "memory");
                }
            };
            const __half2 minus72 = __float2half2_rn(-72.0f);
            int ids = look_up(0), next_ids = look_up(1);
            if (warp < kKWarp0 + kKWarps) {
                constexpr int PER = kTilePages / kKWarps;
                const int kw = warp - kKWarp0;
                uint32_t code[PER][2][WORDS], scale[PER][2][NG / 2];
                auto fetch = [&](int i, int from) {
                    const int id = __shfl_sync(0xffffffffu, from, kw * PER + i);
                    if (id >= 0) {
                        const unsigned char* p = head + id * page_stride;
                        load_words<WORDS>(p + lane * (4 * WORDS), code[i][0]);
                        load_words<WORDS>(p + BLOCK / 2 + lane * (4 * WORDS), code[i][1]);
                        load_words<NG / 2>(p + 16 * HD + g * (2 * NG), scale[i][0]);
                        load_words<NG / 2>(p + 16 * HD + (g + 8) * (2 * NG), scale[i][1]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int u = 0; u < NG / 2; ++u) scale[i][h][u] = 0u;
                        }
                    }
                };
#pragma unroll
                for (int i = 0; i < PER; ++i) fetch(i, ids);
                for (int j = 0; j < n_tiles; ++j) {
                    if (j >= T::K_SLOTS) wait(k_empty + 8 * (j % T::K_SLOTS), j / T::K_SLOTS - 1);
                    const uint32_t to = at + T::K_AT + (j % T::K_SLOTS) * T::K_TILE + t * T::K_STRIDE + (4 * (g >> 1) + (g & 1)) * 16;
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int G = 0; G < NG; ++G) {
                                const __half2 s = as_half2(__byte_perm(scale[i][h][G >> 1], 0u, (G & 1) ? 0x3232u : 0x1010u));
                                uint32_t y[4];
                                word_values(code[i][h][G], s, __hmul2(s, minus72), y);
                                sts128(to + 4 * G * T::K_STRIDE + ((kw * PER + i) * kQ4Page + 2 * h) * 16, make_uint4(y[0], y[1], y[2], y[3]));
                            }
                        }
                        fetch(i, next_ids);
                    }
                    landed(k_full + 8 * (j % T::K_SLOTS));
                    next_ids = look_up(j + 2);
                }
            } else {
                constexpr int PER = (kTilePages + kVWarps - 1) / kVWarps;
                const int vw = warp - kVWarp0;
                uint32_t code[PER][2][WORDS], scale[PER][2][NG];
                auto fetch = [&](int i, int from) {
                    const int page = vw + i * kVWarps, id = __shfl_sync(0xffffffffu, from, page & 7);
                    if (page < kTilePages && id >= 0) {
                        const unsigned char* p = head + id * page_stride;
                        load_words<WORDS>(p + 8 * HD + lane * (4 * WORDS), code[i][0]);
                        load_words<WORDS>(p + 8 * HD + BLOCK / 2 + lane * (4 * WORDS), code[i][1]);
                        load_words<NG>(p + 17 * HD + t * (4 * NG), scale[i][0]);
                        load_words<NG>(p + 17 * HD + (4 + t) * (4 * NG), scale[i][1]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int u = 0; u < NG; ++u) scale[i][h][u] = 0u;
                        }
                    }
                };
#pragma unroll
                for (int i = 0; i < PER; ++i) fetch(i, ids);
                for (int j = 0; j < n_tiles; ++j) {
                    if (j >= T::V_SLOTS) wait(v_empty + 8 * (j % T::V_SLOTS), j / T::V_SLOTS - 1);
                    const int key0 = (first_tile + j) * kKeys;
                    const bool edge = key0 < low || key0 + kKeys > high;   // what lies where no row looks may be anything
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        const int page = vw + i * kVWarps;
                        if (page < kTilePages) {
                            if (edge) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int k = key0 + page * kQ4Page + 8 * h + 2 * t;
                                    const uint32_t keep = (k >= low && k < high ? 0xffffu : 0u) | (k + 1 >= low && k + 1 < high ? 0xffff0000u : 0u);
#pragma unroll
                                    for (int G = 0; G < NG; ++G) scale[i][h][G] &= keep;
                                }
                            }
                            const uint32_t to = at + T::V_AT + (j % T::V_SLOTS) * T::V_TILE + (2 * page + (t >> 1)) * T::V_STRIDE + g * 16 + (t & 1) * 8;
#pragma unroll
                            for (int G = 0; G < NG; ++G) {
                                uint32_t y0[4], y1[4];
                                const __half2 s0 = as_half2(scale[i][0][G]), s1 = as_half2(scale[i][1][G]);
                                word_values(code[i][0][G], s0, __hmul2(s0, minus72), y0);
                                word_values(code[i][1][G], s1, __hmul2(s1, minus72), y1);
#pragma unroll
                                for (int u = 0; u < 4; ++u) sts64(to + (32 * G + 8 * u) * 16, y0[u], y1[u]);
                            }
                        }
                        fetch(i, next_ids);
                    }
                    landed(v_full + 8 * (j % T::V_SLOTS));
                    next_ids = look_up(j + 2);
                }
            }
        }
    } else {
        // ---------------- softmax: one row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::SOFTMAX_REGS));
        const int t = warp >> 2, row0 = (warp & 3) * 32, row = row0 + lane, flat0 = w.flat0 + t * kRows;
        const uint32_t q_tile = at + T::PLANES * t * T::Q_TILE;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (alive) alive = mbar_wait(bar, parity & 1u, nullptr, 0, kSpinLimit);
        };
        float factor = 0.0f;   // of this thread's row's scores
        if (n[t] > 0) {
            // the warp's 32 query rows: lane = (row of eight, 8-dimension piece of four), scaled so that a row's largest lies in [2^13, 2^14)
            const int sub = lane & 7, pc = lane >> 3;
            constexpr int PP = HD / 32;   // pieces per lane and row
#pragma unroll 1
            for (int rg = 0; rg < 4; ++rg) {
                const int r = row0 + rg * 8 + sub;
                float x[PP][8], top = 0.0f;
#pragma unroll
                for (int p = 0; p < PP; ++p) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[p][i] = 0.0f;
                    if (r < live[t]) q4_load8(a.q, (w.row0 + (flat0 + r) / group) * a.q_stride + (long long)(kvh * group + (flat0 + r) % group) * HD + (p * 4 + pc) * 8, a.type, a.vector_q, x[p]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[p][i]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const int e = top > 0.0f && top < INFINITY ? max(-126, min(126, 140 - (int)(__float_as_uint(top) >> 23))) : 0;
                const float up = __int_as_float((e + 127) << 23), f = __int_as_float((127 - e) << 23), sign = a.scale < 0.0f ? -1.0f : 1.0f;
                const float mine = __shfl_sync(0xffffffffu, f, lane & 7);
                if ((lane >> 3) == rg) factor = mine * (fabsf(a.scale) * kLog2e);
#pragma unroll
                for (int p = 0; p < PP; ++p) {
                    uint4 hi, lo;
                    uint32_t *h = &hi.x, *l = &lo.x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) split2(x[p][i] * up * sign, x[p][i + 4] * up * sign, h[i], l[i]);
                    const uint32_t to = q_tile + (p * 4 + pc) * T::Q_STRIDE + r * 16;
                    sts128(to, hi);
                    if (PAIR) sts128(to + T::Q_TILE, lo);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * t);
        }
        const bool have = row < live[t];
        const int limit = have ? w.base + (flat0 + row) / group : -1, lowest = a.window > 0 ? limit - a.window + 1 : 0;
        // keys that every row of the warp sees
        const int all_high = __reduce_min_sync(0xffffffffu, limit), all_low = __reduce_max_sync(0xffffffffu, lowest);
        const uint32_t lanes = (uint32_t)row0 << 16, s_at = tmem + lanes + 128 * t, o_at = s_at + 256;
        float m = -INFINITY;
        float2 l = make_float2(0.0f, 0.0f);
        float sum[PAIR ? HD : 1], since = 1.0f;   // earlier windows' results; the factor that has come to them since the last one's end
#pragma unroll
        for (int i = 0; i < (PAIR ? HD : 1); ++i) sum[i] = 0.0f;
        auto look_up = [&](int j) -> bool {   // whether page `lane & 7` of tile j lies outside of the arena
            const int p = (first_tile + j) * kTilePages + (lane & 7);
            const int id = j < n[t] && p < table_pages ? table[p] : 0;
            return id < 0 || id >= a.pages;
        };
        bool next_bad = n[t] > 0 && look_up(0);
        for (int j = 0; j < n[t]; ++j) {
            const uint32_t bad = __ballot_sync(0xffffffffu, next_bad) & 0xffu;
            next_bad = look_up(j + 1);
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
            float mx = -INFINITY;
#pragma unroll 1
            for (int i = 0; i < kKeys; i += 32) {
                float s[32];
                tmem_ld32(s_at + i, s);
                tmem_wait_ld();
                tmem_tie32(s);
                if (masked) hide(s, i);
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int u = 4; u < 28; u += 8) {
#pragma unroll
                    for (int v = 0; v < 4; ++v) top[v] = fmaxf(top[v], fmaxf(s[u + v], s[u + 4 + v]));
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) top[v] = fmaxf(top[v], s[28 + v]);
                mx = fmaxf(mx, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
            }
            const bool moves = mx > m && (m == -INFINITY || (mx - m) * factor > kSlack);
            if (__any_sync(0xffffffffu, moves)) {
                const float f = moves ? (m == -INFINITY ? 0.0f : exp2_approx((m - mx) * factor)) : 1.0f;
                if (moves) m = mx;
                l.x *= f; l.y *= f;
                if (PAIR) since *= f;
                if (!fresh) {
#pragma unroll 1
                    for (int i = 0; i < HD; i += 16) {
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
                }
            }
            const float shift = m == -INFINITY ? 0.0f : kHeld - m * factor;
#pragma unroll 1
            for (int i = 0; i < kKeys; i += 32) {
                float s[32];
                tmem_ld32(s_at + i, s);
                tmem_wait_ld();
                tmem_tie32(s);
                if (masked) hide(s, i);
                uint32_t hi[16], lo[PAIR ? 16 : 1];
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const float2 x = __ffma2_rn(make_float2(s[2 * u], s[2 * u + 1]), make_float2(factor, factor), make_float2(shift, shift));
                    const float2 p = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    l = __fadd2_rn(l, p);
                    if (PAIR) split2(p.x, p.y, hi[u], lo[PAIR ? u : 0]);
                    else hi[u] = as_bits(__floats2half2_rn(p.x, p.y));
                }
                tmem_st16(s_at + i, hi);   // over the 32 scores just read
                if constexpr (PAIR) tmem_st16(s_at + i + 16, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * t);
        }
        if (n[t] > 0) {
            wait(o_full + 8 * t, 0);
            tc_fence_after();
        }
        // rows to memory through the shared memory that the queries have left: a warp's own rows, in 16-byte pieces by number ^ (row % 8)
        if (live[t] > row0) {
            constexpr int VALUE = PAIR ? 4 : 2, ROW_BYTES = HD * VALUE, PIECES = ROW_BYTES / 16;
            const float total = l.x + l.y;
            const uint32_t stage = q_tile + row0 * ROW_BYTES;
            float inv = total > 0.0f ? 1.0f / total : total != total ? total : 0.0f;
            if (!alive || lds32(failed) != 0) inv = __int_as_float(0x7fffffff);
            if (n[t] > 0) {
#pragma unroll
                for (int i = 0; i < HD; i += 32) {
                    float o[32];
                    tmem_ld32(o_at + i, o);
                    tmem_wait_ld();
                    tmem_tie32(o);
#pragma unroll
                    for (int u = 0; u < 32; ++u) {
                        if (PAIR) o[u] = fmaf(sum[PAIR ? i + u : 0], since, o[u]);
                        o[u] = total > 0.0f || total != total ? o[u] * inv : 0.0f;
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
                        sts128(stage + lane * ROW_BYTES + ((((i + u) * VALUE / 16) ^ (lane & 7)) << 4), v);
                    }
                }
            } else {   // no key for any row of the tile
#pragma unroll
                for (int i = 0; i < PIECES; ++i) sts128(stage + lane * ROW_BYTES + (i << 4), make_uint4(0u, 0u, 0u, 0u));
            }
            __syncwarp();
            constexpr int PER = 32 / PIECES;   // rows per pass
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += PER) {
                const int r = r0 + lane / PIECES, p = lane % PIECES, flat = flat0 + row0 + r;
                if (row0 + r >= live[t]) continue;
                const uint4 v = lds128(stage + r * ROW_BYTES + ((p ^ (r & 7)) << 4));
                const long long to = (w.row0 + flat / group) * a.out_stride + (long long)(kvh * group + flat % group) * HD + p * (16 / VALUE);
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
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int HD, bool PAIR>
cudaError_t launch_tile(cudaStream_t stream, const KvQ4Attention& a) {
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
    const long long flats = (long long)a.rows * (a.q_heads / a.kv_heads);
    const long long places = flats / (2 * kRows) + std::min<long long>(a.sequences, flats / (a.tile_above + 1));
    if (places * a.kv_heads > 0x7fffffffll) return cudaErrorInvalidValue;
    if (places <= 0) return cudaSuccess;
    kvq4_tile_kernel<HD, PAIR><<<(unsigned)(places * a.kv_heads), kThreads, Tile<HD, PAIR>::SMEM, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kvq4_tiles(cudaStream_t stream, const KvQ4Attention& a) {
    const bool pair = a.type == kQ4F32;
    if (a.head_dim == 64) return pair ? launch_tile<64, true>(stream, a) : launch_tile<64, false>(stream, a);
    if (a.head_dim == 128) return pair ? launch_tile<128, true>(stream, a) : launch_tile<128, false>(stream, a);
    return cudaErrorInvalidValue;
}

}  // namespace ribn
