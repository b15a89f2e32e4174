// Writing rows into the 4-bit KV cache (kvq4.cuh) and reading them back.
//
// A thread has eight neighbouring dimensions of one row's K or V, the four threads of a group of 32 together its value x of
// largest magnitude (of several the first).  scale = x / -8 as binary16, then rounded to seven significant bits, half away from
// zero, at most 896 in magnitude; code = clamp(floor(value / scale + 1/2), -8, 7) + 8.  The quotient is formed with a reciprocal
// and its remainder, which a fused multiply-add gives exactly here (seven-bit scale, quotient of four bits), decides the code:
// it is the one that exact arithmetic gives.  NaN counts as zero, infinities as the largest value.
#include <math.h>

#include "kvq4.cuh"

namespace ribn {

namespace {

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

// Where a row's eight dimensions lie: piece p of head_dim / 8.
struct Piece {
    long long row;
    int head, which, p;   // which: 0 K, 1 V
};
__device__ __forceinline__ Piece piece_of(long long id, int kv_heads, int pieces) {
    Piece r;
    r.p = (int)(id % pieces);
    const long long rest = id / pieces;
    r.head = (int)(rest % kv_heads);
    const long long more = rest / kv_heads;
    r.which = (int)(more & 1);
    r.row = more >> 1;
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

template <int TYPE>
__global__ void __launch_bounds__(256) kvq4_append_kernel(const KvQ4Rows a, const bool vector) {
    const int pieces = a.head_dim / 8, lane = threadIdx.x & 31;
    const long long total = a.rows * a.kv_heads * 2 * pieces;   // a multiple of eight: groups of four lanes stay whole
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool inside = id < total;
    const Piece at = piece_of(inside ? id : 0, a.kv_heads, pieces);
    const long long slot = a.slots[at.row];
    const bool live = inside && slot >= 0 && slot < a.pages * kQ4Page;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (live) q4_load8<TYPE == kQ4F32>(at.which ? a.v : a.k, at.row * (at.which ? a.v_stride : a.k_stride) + (long long)at.head * a.head_dim + at.p * 8, TYPE, vector, x);
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
    const uint32_t size = min(((raw & 0x7fffu) + 8u) & ~15u, 0x6300u), scale_bits = size | (raw & 0x8000u);
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
    const int i4 = at.p & 3, G = at.p >> 2;
    const uint32_t halves = gather_nibbles(word, i4, lane);
    if (!live) return;
    const int j = (int)(slot & (kQ4Page - 1));
    unsigned char* record = a.cache + ((slot >> 4) * a.kv_heads + at.head) * q4_record(a.head_dim);
    if (at.which == 0) {
        *reinterpret_cast<uint32_t*>(record + k_word_at(a.head_dim, j, at.p)) = word;
        if (i4 == 0) *reinterpret_cast<unsigned short*>(record + k_scale_at(a.head_dim, j, G)) = (unsigned short)scale_bits;
    } else {
        *reinterpret_cast<unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4)) = (unsigned short)halves;
        *reinterpret_cast<unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4 + 1)) = (unsigned short)(halves >> 16);
        if (i4 == 0) *reinterpret_cast<unsigned short*>(record + v_scale_at(a.head_dim, j, G)) = (unsigned short)scale_bits;
    }
}

template <int TYPE>
__global__ void __launch_bounds__(256) kvq4_read_kernel(const KvQ4Rows a) {
    const int pieces = a.head_dim / 8, lane = threadIdx.x & 31;
    const long long total = a.rows * a.kv_heads * 2 * pieces;
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool inside = id < total;
    const Piece at = piece_of(inside ? id : 0, a.kv_heads, pieces);
    const long long slot = a.slots[at.row];
    const bool live = inside && slot >= 0 && slot < a.pages * kQ4Page;
    const int i4 = at.p & 3, G = at.p >> 2, j = (int)(slot & (kQ4Page - 1));
    const unsigned char* record = a.cache + (live ? ((slot >> 4) * a.kv_heads + at.head) * q4_record(a.head_dim) : 0);
    uint32_t word = 0x88888888u, scale = 0;
    if (live) {
        if (at.which == 0) {
            word = *reinterpret_cast<const uint32_t*>(record + k_word_at(a.head_dim, j, at.p));
            scale = *reinterpret_cast<const unsigned short*>(record + k_scale_at(a.head_dim, j, G));
        } else {
            word = (uint32_t)*reinterpret_cast<const unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4)) |
                   (uint32_t)*reinterpret_cast<const unsigned short*>(record + v_word_at(a.head_dim, j, G, 2 * i4 + 1)) << 16;
            scale = *reinterpret_cast<const unsigned short*>(record + v_scale_at(a.head_dim, j, G));
        }
    }
    const uint32_t back = scatter_nibbles(word, i4, lane);
    if (at.which != 0) word = back;
    const __half2 s = __half2half2(__ushort_as_half((unsigned short)scale)), shift = __float2half2_rn(1032.0f);
    __half2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // 1024 + code, exact
        const uint32_t pair = 0x64006400u | ((word >> (8 * i)) & 15u) | ((word >> (8 * i + 4)) & 15u) << 16;
        x[i] = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&pair), shift), s);
    }
    if (inside) store8<TYPE>(const_cast<void*>(at.which ? a.v : a.k), at.row * (at.which ? a.v_stride : a.k_stride) + (long long)at.head * a.head_dim + at.p * 8, x);
}

bool aligned16(const void* p, long long stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; }

}  // namespace

cudaError_t launch_kvq4_append(cudaStream_t stream, const KvQ4Rows& a) {
    if (a.rows <= 0) return cudaSuccess;
    const long long threads = a.rows * a.kv_heads * 2 * (a.head_dim / 8), blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    const int size = a.type == kQ4F32 ? 4 : 2;
    const bool vector = aligned16(a.k, a.k_stride, size) && aligned16(a.v, a.v_stride, size);
    if (a.type == kQ4F32) kvq4_append_kernel<kQ4F32><<<(unsigned)blocks, 256, 0, stream>>>(a, vector);
    else if (a.type == kQ4F16) kvq4_append_kernel<kQ4F16><<<(unsigned)blocks, 256, 0, stream>>>(a, vector);
    else kvq4_append_kernel<kQ4BF16><<<(unsigned)blocks, 256, 0, stream>>>(a, vector);
    return cudaGetLastError();
}

cudaError_t launch_kvq4_read(cudaStream_t stream, const KvQ4Rows& a) {
    if (a.rows <= 0) return cudaSuccess;
    const long long threads = a.rows * a.kv_heads * 2 * (a.head_dim / 8), blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    if (a.type == kQ4F32) kvq4_read_kernel<kQ4F32><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else if (a.type == kQ4F16) kvq4_read_kernel<kQ4F16><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else kvq4_read_kernel<kQ4BF16><<<(unsigned)blocks, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace ribn
