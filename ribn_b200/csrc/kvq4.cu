// Writing rows into the 4-bit KV cache (kvq4.cuh) and reading them back.
//
// A thread has eight neighbouring dimensions of one row's K or V, the four threads of a group of 32 together its value x of
// largest magnitude (of several the first).  scale = x / -8 as binary16, then rounded to seven significant bits, half away from
// zero, at most 896 in magnitude; code = clamp(floor(value / scale + 1/2), -8, 7) + 8.  The quotient is formed with a reciprocal
// and its remainder, which a fused multiply-add gives exactly here (seven-bit scale, quotient of four bits), decides the code:
// it is the one that exact arithmetic gives.  NaN counts as zero, infinities as the largest value.
//
// What bounds it: reading 60,001 rows (8 heads of 128) back as F32 moves 561 MB in 100 us, 84 % of the copy bandwidth (134 us with one
// row a thread); 16,384 as F16 86 MB in 27 us.  Writing 2,048 BF16 rows takes 10 us for 11 MB, the quantiser's instructions (7.4 M
// of warps, the logic pipe 76 % busy).  A row of V
// is written as half words because a word belongs to two tokens.  Short calls are a launch.
#include <math.h>

#include "kvq4.cuh"

namespace ribn {

namespace {

constexpr unsigned kRowThreads = 256;

__device__ __forceinline__ uint32_t bits_of(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// Eight values that binary16 holds exactly
template <int TYPE>
__device__ __forceinline__ void store8(void* base, long long at, const __half2 (&x)[4]) {
    if (TYPE == kQ4F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        const float2 a = __half22float2(x[0]), b = __half22float2(x[1]), c = __half22float2(x[2]), d = __half22float2(x[3]);
        p[0] = make_float4(a.x, a.y, b.x, b.y);
        p[1] = make_float4(c.x, c.y, d.x, d.y);
    } else {
        uint4 w;
        uint32_t* o = &w.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (TYPE == kQ4F16) {
                o[i] = bits_of(x[i]);
            } else {   // the type asked for has eight bits where the value has eleven: rounded to the nearest
                const float2 f = __half22float2(x[i]);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(f.y), "f"(f.x));
            }
        }
        *reinterpret_cast<uint4*>(static_cast<unsigned short*>(base) + at) = w;
    }
}

// Where a thread's eight dimensions lie: piece p of head_dim / 8 of `many` rows, `row` the first and `step` from one to the next.  A block
// has `many` times some rows, or 256 pieces of as many.  Calls with many rows give a thread four, whose loads travel together.
struct Piece {
    long long row, step;
    int head, which, p;   // which: 0 K, 1 V
    bool inside;
};
__device__ __forceinline__ Piece piece_of(const KvQ4Rows& a, int many) {
    // (32-bit arithmetic throughout: with three 64-bit divisions a thread 16,384 rows took 37 us to read back)
    const int log_pieces = a.head_dim == 64 ? 3 : a.head_dim == 128 ? 4 : 5;
    const unsigned per_row = (unsigned)(2 * a.kv_heads) << log_pieces;
    Piece r;
    unsigned rest;
    if (per_row <= kRowThreads) {
        const unsigned rows = kRowThreads / per_row, mine = threadIdx.x / per_row;
        r.row = (long long)blockIdx.x * rows * many + mine;
        r.step = rows;
        rest = threadIdx.x - mine * per_row;
        r.inside = mine < rows;
    } else {
        const unsigned blocks = (per_row + kRowThreads - 1) / kRowThreads, row = blockIdx.x / blocks;
        r.row = (long long)row * many;
        r.step = 1;
        rest = (blockIdx.x - row * blocks) * kRowThreads + threadIdx.x;
        r.inside = rest < per_row;
    }
    if (!r.inside) rest = 0;
    r.p = (int)(rest & ((1u << log_pieces) - 1));
    const unsigned more = rest >> log_pieces;
    r.which = more >= (unsigned)a.kv_heads;
    r.head = (int)(r.which ? more - (unsigned)a.kv_heads : more);
    return r;
}

// The word of K codes, and the scale, of piece p (group G = p / 4, quarter t = p % 4) of token j
__device__ __forceinline__ int k_word_at(int head_dim, int j, int p) {
    const int words = head_dim == 64 ? 2 : 4, G = p >> 2;
    return (G / words) * (kQ4Page * 16 * words) + j * (16 * words) + (p & 3) * (4 * words) + (G % words) * 4;
}
__device__ __forceinline__ int k_scale_at(int head_dim, int j, int G) { return 16 * head_dim + (j * (head_dim / 32) + G) * 2; }
// The half word of V codes of dimensions 32 G + g + {0, 8, 16, 24}
__device__ __forceinline__ int v_word_at(int head_dim, int j, int G, int g) {
    const int words = head_dim == 64 ? 2 : 4;
    return 8 * head_dim + (G / words) * (kQ4Page * 16 * words) + (j >> 3) * (128 * words) + g * (16 * words) + ((j >> 1) & 3) * (4 * words) +
           (G % words) * 4 + (j & 1) * 2;
}
__device__ __forceinline__ int v_scale_at(int head_dim, int j, int G) {
    return 17 * head_dim + (((j >> 1) * (head_dim / 32) + G) * 2 + (j & 1)) * 2;
}

// Nibble transposition within four lanes (p % 4 = i): lane i has word_i with a nibble per g; it gets the half words of g = 2 i
// (low) and 2 i + 1 (high), nibble i' from word_i'.  Its own inverse but for the packing.
__device__ __forceinline__ uint32_t gather_nibbles(uint32_t word, int i, int lane) {
    uint32_t r = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const uint32_t w = __shfl_sync(0xffffffffu, word, (lane & ~3) + u) >> (8 * i);
        r |= (w & 15u) << (4 * u) | ((w >> 4) & 15u) << (16 + 4 * u);
    }
    return r;
}
__device__ __forceinline__ uint32_t scatter_nibbles(uint32_t halves, int i, int lane) {
    uint32_t r = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {   // lane u has the half words of g = 2 u and 2 u + 1
        const uint32_t w = __shfl_sync(0xffffffffu, halves, (lane & ~3) + u) >> (4 * i);
        r |= (w & 15u) << (8 * u) | ((w >> 16) & 15u) << (8 * u + 4);
    }
    return r;
}

// The word of codes (nibble i: value i) of a thread's eight values and the scale of its group's 32, which four neighbouring threads have
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], int lane, uint32_t& scale_bits) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (x[i] != x[i]) x[i] = 0.0f;
        if (fabsf(x[i]) > fabsf(top)) top = x[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {   // the lower lane's value stands where both are as large
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        const float low = (lane & o) ? other : top, high = (lane & o) ? top : other;
        top = fabsf(high) > fabsf(low) ? high : low;
    }
    const uint32_t raw = __half_as_ushort(__float2half_rn(top * -0.125f));
    const uint32_t size = min(((raw & 0x7fffu) + 8u) & ~15u, 0x6300u);
    scale_bits = size | (raw & 0x8000u);
    const float d = __half2float(__ushort_as_half((unsigned short)size)), inv = d > 0.0f ? 1.0f / d : 0.0f, half = 0.5f * d;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = __uint_as_float(__float_as_uint(x[i]) ^ ((raw & 0x8000u) << 16));
        float q = floorf(fminf(fmaxf(y * inv, -9.0f), 9.0f) + 0.5f);
        const float rest = fmaf(-q, d, y);
        q += d > 0.0f ? (rest >= half ? 1.0f : rest < -half ? -1.0f : 0.0f) : 0.0f;
        word |= (uint32_t)((int)fminf(fmaxf(q, -8.0f), 7.0f) + 8) << (4 * i);
    }
    return word;
}

template <int TYPE, int MANY>
__global__ void __launch_bounds__(kRowThreads) kvq4_append_kernel(const KvQ4Rows a, const bool vector) {
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Piece at = piece_of(a, MANY);   // a row has a multiple of eight: groups of four lanes are of one group of dimensions
    constexpr int WORDS = TYPE == kQ4F32 ? 8 : 4;
    uint32_t raw[MANY][WORDS];
    int slot[MANY];
#pragma unroll
    for (int u = 0; u < MANY; ++u) {
        const long long row = at.row + u * at.step;
        const bool inside = at.inside && row < a.rows;
        slot[u] = inside ? a.slots[row] : -1;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) raw[u][i] = 0u;
        if (inside) q4_load_raw(at.which ? a.v : a.k, row * (at.which ? a.v_stride : a.k_stride) + (long long)at.head * a.head_dim + at.p * 8, vector, raw[u]);
    }
    const int i4 = lane & 3, G = at.p >> 2;
#pragma unroll
    for (int u = 0; u < MANY; ++u) {
        float x[8];
        q4_values(raw[u], TYPE, x);
        uint32_t scale_bits;
        const uint32_t word = quantise8(x, lane, scale_bits), halves = gather_nibbles(word, i4, lane);
        if (slot[u] < 0 || slot[u] >= a.pages * kQ4Page) continue;   // (the shuffles above are done)
        const int j = slot[u] & (kQ4Page - 1);
        unsigned char* record = a.cache + ((long long)(slot[u] >> 4) * a.kv_heads + at.head) * q4_record(a.head_dim);
        if (at.which == 0) {
            *reinterpret_cast<uint32_t*>(record + k_word_at(a.head_dim, j, at.p)) = word;
            if (i4 == 0) *reinterpret_cast<unsigned short*>(record + k_scale_at(a.head_dim, j, G)) = (unsigned short)scale_bits;
        } else {
            *reinterpret_cast<unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4)) = (unsigned short)halves;
            *reinterpret_cast<unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4 + 1)) = (unsigned short)(halves >> 16);
            if (i4 == 0) *reinterpret_cast<unsigned short*>(record + v_scale_at(a.head_dim, j, G)) = (unsigned short)scale_bits;
        }
    }
}

template <int TYPE, int MANY>
__global__ void __launch_bounds__(kRowThreads) kvq4_read_kernel(const KvQ4Rows a) {
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Piece at = piece_of(a, MANY);
    const int i4 = lane & 3, G = at.p >> 2;
    int slot[MANY];
    uint32_t word[MANY], scale[MANY];
#pragma unroll
    for (int u = 0; u < MANY; ++u) {
        const long long row = at.row + u * at.step;
        slot[u] = at.inside && row < a.rows ? a.slots[row] : -1;
    }
#pragma unroll
    for (int u = 0; u < MANY; ++u) {
        const int j = slot[u] & (kQ4Page - 1);
        word[u] = 0x88888888u;
        scale[u] = 0;
        if (slot[u] >= 0 && slot[u] < a.pages * kQ4Page) {
            const unsigned char* record = a.cache + ((long long)(slot[u] >> 4) * a.kv_heads + at.head) * q4_record(a.head_dim);
            if (at.which == 0) {
                word[u] = *reinterpret_cast<const uint32_t*>(record + k_word_at(a.head_dim, j, at.p));
                scale[u] = *reinterpret_cast<const unsigned short*>(record + k_scale_at(a.head_dim, j, G));
            } else {
                word[u] = (uint32_t)*reinterpret_cast<const unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4)) |
                          (uint32_t)*reinterpret_cast<const unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4 + 1)) << 16;
                scale[u] = *reinterpret_cast<const unsigned short*>(record + v_scale_at(a.head_dim, j, G));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < MANY; ++u) {
        const uint32_t back = scatter_nibbles(word[u], i4, lane), w = at.which ? back : word[u];
        const __half2 s = __half2half2(__ushort_as_half((unsigned short)scale[u])), shift = __float2half2_rn(1032.0f);
        __half2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // 1024 + code, exact
            const uint32_t pair = 0x64006400u | ((w >> (8 * i)) & 15u) | ((w >> (8 * i + 4)) & 15u) << 16;
            x[i] = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&pair), shift), s);
        }
        const long long row = at.row + u * at.step;
        if (at.inside && row < a.rows) {
            store8<TYPE>(const_cast<void*>(at.which ? a.v : a.k), row * (at.which ? a.v_stride : a.k_stride) + (long long)at.head * a.head_dim + at.p * 8, x);
        }
    }
}

bool aligned16(const void* p, long long stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; }

// Early launch: the kernel's blocks stand ready when the one before ends (each waits for it before it reads anything).
template <typename Kernel, typename... Args>
cudaError_t launch_rows(cudaStream_t stream, Kernel kernel, const KvQ4Rows& a, int many, Args... more) {
    const long long per_row = 2ll * a.kv_heads * (a.head_dim / 8);
    const long long together = (per_row <= kRowThreads ? kRowThreads / per_row : 1) * many;   // rows of a block
    const long long blocks = (a.rows + together - 1) / together * (per_row <= kRowThreads ? 1 : (per_row + kRowThreads - 1) / kRowThreads);
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, more...);
}
bool many_rows(const KvQ4Rows& a) { return a.rows * a.kv_heads * (a.head_dim / 4) > 2ll * 2048 * kvq4_sm_count(); }

// Four rows a thread where one each would fill the GPU's threads more than twice over
template <int TYPE>
cudaError_t launch_append(cudaStream_t stream, const KvQ4Rows& a, bool vector) {
    return many_rows(a) ? launch_rows(stream, kvq4_append_kernel<TYPE, 4>, a, 4, vector) : launch_rows(stream, kvq4_append_kernel<TYPE, 1>, a, 1, vector);
}
template <int TYPE>
cudaError_t launch_read(cudaStream_t stream, const KvQ4Rows& a) {
    return many_rows(a) ? launch_rows(stream, kvq4_read_kernel<TYPE, 4>, a, 4) : launch_rows(stream, kvq4_read_kernel<TYPE, 1>, a, 1);
}

}  // namespace

cudaError_t launch_kvq4_append(cudaStream_t stream, const KvQ4Rows& a) {
    if (a.rows <= 0) return cudaSuccess;
    const int size = a.type == kQ4F32 ? 4 : 2;
    const bool vector = aligned16(a.k, a.k_stride, size) && aligned16(a.v, a.v_stride, size);
    return a.type == kQ4F32 ? launch_append<kQ4F32>(stream, a, vector) : a.type == kQ4F16 ? launch_append<kQ4F16>(stream, a, vector) : launch_append<kQ4BF16>(stream, a, vector);
}

cudaError_t launch_kvq4_read(cudaStream_t stream, const KvQ4Rows& a) {
    if (a.rows <= 0) return cudaSuccess;
    return a.type == kQ4F32 ? launch_read<kQ4F32>(stream, a) : a.type == kQ4F16 ? launch_read<kQ4F16>(stream, a) : launch_read<kQ4BF16>(stream, a);
}

}  // namespace ribn
