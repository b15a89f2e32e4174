// The KV cache held in 4 bits: layout, arguments of its launchers, and what its kernels share.
//
// The arena is [pages][kv_heads][18 head_dim] bytes, 16 tokens a page: a page of one head is one contiguous record
//   K codes, 8 head_dim bytes   [sub][token j][t][w][4 bytes]       nibble i of a word: dimension 32 G + 8 t + i
//   V codes, 8 head_dim bytes   [sub][c][g][t][w][e][2 bytes]       nibble i of a half word: dimension 32 G + 8 i + g, j = 8 c + 2 t + e
//   K scales, head_dim bytes    [j][G] binary16
//   V scales, head_dim bytes    [c][t][G][e] binary16
// with G = 4 sub + w the group of 32 dimensions (a head of 64 has two: w < 2).  A value is scale x (code - 8).  A scale has seven
// significant bits, so the value (four more) and 72 x scale (four more) are binary16 numbers, without any rounding.
//
// The order is the matrix instructions': of a K page a lane (g = lane / 4, t = lane % 4) reads 16 bytes of keys g and g + 8, of a
// V page 16 bytes of key pairs 2 t and 8 + 2 t, and masks and shifts turn the words into the operands of m16n8k16 with the keys
// (K) or the dimensions (V) as rows.  A byte belongs to one token, so writing a token's row reads nothing.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemv.cuh"

namespace ribn {

constexpr int kQ4Page = 16;            // tokens per page
constexpr int kQ4MaxGroup = 16;        // query heads per kv head
constexpr uint32_t kQ4WaitPolls = 1u << 22;
__host__ __device__ constexpr int q4_record(int head_dim) { return 18 * head_dim; }

enum Q4Type : int { kQ4F32 = 0, kQ4F16 = 1, kQ4BF16 = 2 };

struct KvQ4Rows {
    unsigned char* cache;
    long long pages;
    int kv_heads, head_dim, type;
    const void* k;                     // [rows][kv_heads][head_dim]; written by a read
    const void* v;
    long long k_stride, v_stride;      // values between rows
    const int32_t* slots;              // page * 16 + token; outside of the arena: the row is skipped (append) or zero (read)
    long long rows;
};
cudaError_t launch_kvq4_append(cudaStream_t stream, const KvQ4Rows& a);
cudaError_t launch_kvq4_read(cudaStream_t stream, const KvQ4Rows& a);

struct KvQ4Attention {
    const unsigned char* cache;
    long long pages;
    int q_heads, kv_heads, head_dim, type;
    const void* q;                     // [rows][q_heads][head_dim]
    long long q_stride, out_stride;    // values between rows
    void* out;
    const int32_t* page_tables;        // [sequences][table_stride]
    int pages_per_sequence;
    long long table_stride;
    const int32_t* lengths;            // [sequences] keys, the new rows' among them
    const int32_t* cu_rows;            // [sequences + 1]
    int sequences, rows, max_rows, max_keys, window;
    float scale;                       // of the scores
    uint32_t wait_polls;               // of a barrier in the tile kernel, before the wait has run out
    float* partial;                    // scratch of partial_bytes: the runs' sums and the operands below
    size_t partial_bytes;
    // set by the launcher
    int sms;                           // of the device
    int grid, set_up, span_cols, col_blocks, merge_cols, vector_q, vector_out;
    long long* prefix;                 // pages of the span kernel's list before each sequence, and of all
    unsigned char* scratch;            // operands of the tile kernel's key tiles, [tile][kv_head][512 head_dim bytes]
    int scratch_tiles;                 // how many tiles there is room for
    int tile_splits;                   // CTAs that share a pair of query tiles' keys, their sums in tile_partial, [row][q_head][split][head_dim + 4]
    float* tile_partial;
    int tile_above;                    // a sequence with more query rows (rows x heads of a group) than this takes the tile kernel
};
static_assert(sizeof(KvQ4Attention) <= 224, "with 232 bytes of arguments a launch takes 0.4 us longer on the host");
// Bytes of scratch that launch_kvq4_attention can use; it works with less than the tile kernel's part, not with less than the sums.
// It does not shrink with `sms`, so that asked for kvq4_most_sms() it does on every device.
size_t kvq4_workspace_bytes(const KvQ4Attention& a, int sms);
int kvq4_most_sms();
cudaError_t launch_kvq4_attention(cudaStream_t stream, KvQ4Attention a);

// The sequences with more than `tile_above` query rows (kvq4_tile.cu; heads of 64 and 128).
cudaError_t launch_kvq4_tiles(cudaStream_t stream, const KvQ4Attention& a);
// At most this many pairs of its query tiles, however the rows are spread over the sequences.
long long kvq4_tile_places(const KvQ4Attention& a);

int kvq4_sm_count();

// Sets the calling thread's operator diagnostic (ops_api.cu); returns RIBN_B200_ERROR.
int op_error(const char* what, cudaError_t e);

// Eight neighbouring values of a row as they lie (F32: eight words, else four) ..
template <int WORDS>
__device__ __forceinline__ void q4_load_raw(const void* base, long long at, bool vector, uint32_t (&w)[WORDS]) {
    if (vector) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + at * (WORDS / 2));
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) {
            const uint4 u = p[i];
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
    } else if (WORDS == 8) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = static_cast<const uint32_t*>(base)[at + i];
    } else {
        const unsigned short* p = static_cast<const unsigned short*>(base) + at;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    }
}
// .. and as F32
template <int WORDS>
__device__ __forceinline__ void q4_values(const uint32_t (&w)[WORDS], int type, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if (WORDS == 8) {
            x[i] = __uint_as_float(w[i]);
        } else if (type == kQ4F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[(2 * i) & 7] = f.x; x[(2 * i + 1) & 7] = f.y;
        } else {
            x[(2 * i) & 7] = __uint_as_float(w[i] << 16); x[(2 * i + 1) & 7] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <bool WIDE>
__device__ __forceinline__ void q4_load8(const void* base, long long at, int type, bool vector, float (&x)[8]) {
    uint32_t w[WIDE ? 8 : 4];
    q4_load_raw(base, at, vector, w);
    q4_values(w, type, x);
}

// A row's score factor in base 2, of (2^-e of its queries) x |scale of the scores|, kept where every product with a sum of its scaled queries and
// keys (at most 2^35: 256 x 2^14 x 2^13) is finite, and none with an infinity NaN.  Below 2^-126 all scores are as good as zero either way, above
// 2^92 the largest one has all the weight either way (sums that differ do so by 2^-44 or more, the last bits' product).
__device__ __forceinline__ float q4_factor(float x) { return fminf(fmaxf(x * 1.4426950408889634f, 1.17549435e-38f), 4.9517602e27f); }

}  // namespace ribn
