// C-ABI entry points of the 4-bit KV cache: checks, the device of the call, launches (kvq4.cu, kvq4_attention.cu).
#include <math.h>
#include <string.h>

#include "../../include/ribn_b200.h"
#include "kvq4.cuh"

using namespace ribn;

namespace {

// Why the geometry of an arena is refused, or null.  Slots are 32-bit.
const char* bad_arena(const void* cache, int64_t pages, int32_t kv_heads, int32_t head_dim, int32_t type) {
    if (type != RIBN_B200_KVQ4_F32 && type != RIBN_B200_KVQ4_F16 && type != RIBN_B200_KVQ4_BF16) return "kvq4: unknown type";
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return "kvq4: head_dim must be 64, 128 or 256";
    if (kv_heads <= 0 || kv_heads > 4096) return "kvq4: kv_heads must be 1 .. 4096";
    if (pages <= 0 || pages > (int64_t)INT32_MAX / kQ4Page) return "kvq4: pages must be 1 .. 2^27 - 1";
    if (cache == nullptr || (reinterpret_cast<uintptr_t>(cache) & 15) != 0) return "kvq4: the cache must be a 16-byte aligned device pointer";
    return nullptr;
}
// Of a row type's values
bool misaligned(const void* p, int32_t type) { return (reinterpret_cast<uintptr_t>(p) & (type == RIBN_B200_KVQ4_F32 ? 3 : 1)) != 0; }

// The launch needs `device` current; the caller's own current device is put back.
struct OnDevice {
    int previous = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (device < 0 || device >= kMaxDevices) return;
        if (cudaGetDevice(&previous) != cudaSuccess) previous = -1;
        ok = previous == device || cudaSetDevice(device) == cudaSuccess;
        changed = ok && previous != device;
    }
    ~OnDevice() {
        if (changed && previous >= 0) cudaSetDevice(previous);
    }
    bool changed = false;
};

template <typename Launch>
int on_device(int32_t device, const char* what, Launch launch) {
    OnDevice scope(device);
    if (!scope.ok) return op_error("kvq4: cannot select the CUDA device", cudaSuccess);
    const cudaError_t e = launch();
    return e == cudaSuccess ? RIBN_B200_OK : op_error(what, e);
}

KvQ4Attention attention_of(const ribn_b200_kvq4_attention_args& x) {
    KvQ4Attention a{};
    a.cache = static_cast<const unsigned char*>(x.cache); a.pages = x.pages;
    a.q_heads = x.q_heads; a.kv_heads = x.kv_heads; a.head_dim = x.head_dim; a.type = x.type;
    a.q = x.q; a.q_stride = x.q_stride; a.out_stride = x.out_stride; a.out = x.out;
    a.page_tables = x.page_tables; a.pages_per_sequence = x.pages_per_sequence; a.table_stride = x.table_stride;
    a.lengths = x.lengths; a.cu_rows = x.cu_rows;
    a.sequences = x.sequences; a.rows = x.rows; a.max_rows = x.max_rows; a.max_keys = x.max_keys;
    a.window = x.window >= x.pages_per_sequence * kQ4Page ? 0 : x.window;   // over everything a sequence can have: none
    a.scale = x.scale == 0.0f ? 1.0f / sqrtf((float)x.head_dim) : x.scale;
    a.partial = static_cast<float*>(x.workspace); a.partial_bytes = x.workspace_bytes;
    return a;
}

// What does not depend on pointers
const char* bad_attention(const ribn_b200_kvq4_attention_args& a) {
    if (a.kv_heads <= 0 || a.q_heads <= 0 || a.q_heads % a.kv_heads != 0 || a.q_heads / a.kv_heads > kQ4MaxGroup) {
        return "kvq4_attention: q_heads must be 1 to 16 times kv_heads";
    }
    if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return "kvq4: head_dim must be 64, 128 or 256";
    if (a.rows < 0 || a.sequences < 0 || a.max_rows < 0 || a.max_keys < 0 || a.window < 0 || a.pages_per_sequence < 0) return "kvq4_attention: negative size";
    if ((int64_t)a.rows * a.q_heads > INT32_MAX || a.pages_per_sequence > (1 << 26) || a.max_keys > INT32_MAX - kQ4Page || a.max_rows > a.rows) {
        return "kvq4_attention: rows x q_heads, pages_per_sequence or max_keys too large, or max_rows over rows";
    }
    // the merge's grid: columns of the page-streaming kernel in whole blocks, of which head_dim 64 and 128 have at most 64
    const int64_t all = (int64_t)a.max_rows * (a.q_heads / a.kv_heads), columns = a.head_dim == 256 || all < 64 ? (all + 15) / 16 * 16 : 64;
    if (columns > 0 && (int64_t)a.sequences * a.kv_heads > INT32_MAX / columns) return "kvq4_attention: too many sequences x kv_heads x rows of a sequence";
    return nullptr;
}

int attend(int32_t device, void* stream, const ribn_b200_kvq4_attention_args* args, uint32_t wait_polls) {
    if (args == nullptr) return op_error("kvq4_attention: null argument", cudaSuccess);
    const ribn_b200_kvq4_attention_args& x = *args;
    if (const char* why = bad_arena(x.cache, x.pages, x.kv_heads, x.head_dim, x.type)) return op_error(why, cudaSuccess);
    if (const char* why = bad_attention(x)) return op_error(why, cudaSuccess);
    if (!(fabsf(x.scale) < INFINITY)) return op_error("kvq4_attention: scale must be finite", cudaSuccess);
    if (x.rows == 0 || x.sequences == 0 || x.max_rows == 0) return RIBN_B200_OK;
    if (x.q == nullptr || x.out == nullptr || x.lengths == nullptr || x.cu_rows == nullptr || (x.page_tables == nullptr && x.pages_per_sequence > 0)) {
        return op_error("kvq4_attention: null device pointer", cudaSuccess);
    }
    if (misaligned(x.q, x.type) || misaligned(x.out, x.type)) return op_error("kvq4_attention: q or out is not aligned to its type", cudaSuccess);
    const int64_t width = (int64_t)x.q_heads * x.head_dim;
    if ((x.rows > 1 && (x.q_stride < width || x.out_stride < width)) || x.q_stride < 0 || x.out_stride < 0 ||
        (x.sequences > 1 && x.table_stride < x.pages_per_sequence) || x.table_stride < 0) {
        return op_error("kvq4_attention: a stride below the length of its rows", cudaSuccess);
    }
    if (x.workspace == nullptr && x.workspace_bytes > 0) return op_error("kvq4_attention: null workspace with a size", cudaSuccess);
    if ((reinterpret_cast<uintptr_t>(x.workspace) & 15) != 0) return op_error("kvq4_attention: the workspace must be 16-byte aligned", cudaSuccess);
    return on_device(device, "kvq4_attention", [&]() -> cudaError_t {
        KvQ4Attention a = attention_of(x);
        a.wait_polls = wait_polls;
        return launch_kvq4_attention(static_cast<cudaStream_t>(stream), a);
    });
}

}  // namespace

extern "C" {

int ribn_b200_kvq4_append(int32_t device, void* stream, void* cache, int64_t pages, int32_t kv_heads, int32_t head_dim, int32_t type,
                          const void* k, int64_t k_stride, const void* v, int64_t v_stride, const int32_t* slots, int64_t rows) {
    if (const char* why = bad_arena(cache, pages, kv_heads, head_dim, type)) return op_error(why, cudaSuccess);
    if (rows < 0) return op_error("kvq4_append: negative rows", cudaSuccess);
    if (rows == 0) return RIBN_B200_OK;
    if (k == nullptr || v == nullptr || slots == nullptr) return op_error("kvq4_append: null device pointer", cudaSuccess);
    if (misaligned(k, type) || misaligned(v, type)) return op_error("kvq4_append: k or v is not aligned to its type", cudaSuccess);
    const int64_t width = (int64_t)kv_heads * head_dim;
    if ((rows > 1 && (k_stride < width || v_stride < width)) || k_stride < 0 || v_stride < 0) {
        return op_error("kvq4_append: row strides below kv_heads x head_dim", cudaSuccess);
    }
    const KvQ4Rows a{static_cast<unsigned char*>(cache), pages, kv_heads, head_dim, type, k, v, k_stride, v_stride, slots, rows};
    return on_device(device, "kvq4_append", [&] { return launch_kvq4_append(static_cast<cudaStream_t>(stream), a); });
}

int ribn_b200_kvq4_read(int32_t device, void* stream, const void* cache, int64_t pages, int32_t kv_heads, int32_t head_dim, int32_t type,
                        const int32_t* slots, int64_t rows, void* k, void* v) {
    if (const char* why = bad_arena(cache, pages, kv_heads, head_dim, type)) return op_error(why, cudaSuccess);
    if (rows < 0) return op_error("kvq4_read: negative rows", cudaSuccess);
    if (rows == 0) return RIBN_B200_OK;
    if (k == nullptr || v == nullptr || slots == nullptr) return op_error("kvq4_read: null device pointer", cudaSuccess);
    if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0) return op_error("kvq4_read: k and v must be 16-byte aligned", cudaSuccess);
    const int64_t width = (int64_t)kv_heads * head_dim;
    const KvQ4Rows a{static_cast<unsigned char*>(const_cast<void*>(cache)), pages, kv_heads, head_dim, type, k, v, width, width, slots, rows};
    return on_device(device, "kvq4_read", [&] { return launch_kvq4_read(static_cast<cudaStream_t>(stream), a); });
}

size_t ribn_b200_kvq4_workspace(const ribn_b200_kvq4_attention_args* args) {
    if (args == nullptr || bad_attention(*args) != nullptr || args->rows == 0 || args->sequences == 0 || args->max_rows == 0) return 0;
    static const int most_sms = kvq4_most_sms();
    return kvq4_workspace_bytes(attention_of(*args), most_sms);
}

int ribn_b200_kvq4_attention(int32_t device, void* stream, const ribn_b200_kvq4_attention_args* args) {
    return attend(device, stream, args, kQ4WaitPolls);
}

size_t ribn_b200_debug_kvq4_workspace(const ribn_b200_kvq4_attention_args* args, int32_t sms) {
    if (args == nullptr || bad_attention(*args) != nullptr || args->rows == 0 || args->sequences == 0 || args->max_rows == 0 || sms < 1) return 0;
    return kvq4_workspace_bytes(attention_of(*args), sms);
}

int ribn_b200_debug_kvq4_attention(int32_t device, void* stream, const ribn_b200_kvq4_attention_args* args, uint32_t wait_polls) {
    return attend(device, stream, args, wait_polls < kQ4WaitPolls ? wait_polls : kQ4WaitPolls);
}

}  // extern "C"
