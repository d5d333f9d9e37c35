// Store into and load from a paged KV cache of microscaled elements (mx_format.h), gfx950.
//
// Both are bound by memory.  Store: one lane per 8 elements of a K row and of a V row (16-byte loads); a block of 32 elements
// is four neighbouring lanes, which agree on its largest magnitude in two lane permutations, so that codes and scales
// are written in the same pass that reads the rows.  Load: one lane per 8 elements as well, 16-byte stores of bf16.
// Measured: 16385 rows of 32 heads of 128 stored as E4M3 in 76 us (5.3 TB/s, what a large copy reaches); 256 rows of 4 heads in 7.1 us (the
// launch); 64 sequences of 256 to 2048 E4M3 rows of 4 heads loaded in 62 us
// (4.2 TB/s; 42 us when the same tensors are loaded again).  The load writes twice what it reads, or more, and past L2: written through it, the same
// took 66 us (65 again), and 3 sequences of 9000 to 33000 E2M1 rows with the store of 5 before them 37 us instead of 23.  More chunks in flight per
// thread gained nothing.
#include "mx_format.h"

namespace dfx {
namespace {

constexpr int kThreads = 256;

DFX_D int64_t index_at(const void* p, int64_t i, int type) {
    return type == DFX_INDEX_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// ---------------------------------------------------------------- store
struct MxStoreArgs {
    const uint16_t* key;
    const uint16_t* value;
    int64_t key_stride, value_stride;
    uint8_t* k_cache;
    uint8_t* v_cache;
    uint8_t* k_scales;
    uint8_t* v_scales;
    const void* slots;
    int64_t n_tokens, n_slots;
    int slot_type, row_chunks;  // 8-element chunks of a token row (all heads)
};

template <bool E2M1>
__global__ void __launch_bounds__(kThreads) mx_store_kernel(const MxStoreArgs a) {
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (idx >= a.n_tokens * a.row_chunks) return;  // (whole quads: row_chunks is a multiple of 4)
    int64_t t;
    int c;
    if (a.n_tokens * a.row_chunks <= UINT32_MAX) {  // (a 64-bit division costs more than the rest of the kernel)
        const uint32_t i = static_cast<uint32_t>(idx), q = i / static_cast<uint32_t>(a.row_chunks);
        t = q;
        c = static_cast<int>(i - q * static_cast<uint32_t>(a.row_chunks));
    } else {
        t = idx / a.row_chunks;
        c = static_cast<int>(idx - t * a.row_chunks);
    }
    const int64_t slot = index_at(a.slots, t, a.slot_type);
    if (slot < 0 || slot >= a.n_slots) return;
    const u32x4 k8 = *reinterpret_cast<const u32x4*>(a.key + t * a.key_stride + c * 8);
    const u32x4 v8 = *reinterpret_cast<const u32x4*>(a.value + t * a.value_stride + c * 8);
    const int64_t row = slot * a.row_chunks * (E2M1 ? 4 : 8), srow = slot * (a.row_chunks >> 2);
    const bool leads = (c & 3) == 0;
    mx_put8<E2M1>(k8, max_quad(abs_max8(k8)), a.k_cache + row, a.k_scales + srow, c, leads);
    mx_put8<E2M1>(v8, max_quad(abs_max8(v8)), a.v_cache + row, a.v_scales + srow, c, leads);
}

// ---------------------------------------------------------------- load
struct MxLoadArgs {
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    const uint16_t* k_new;
    const uint16_t* v_new;
    int64_t k_new_stride, v_new_stride;
    uint16_t* k_out;
    uint16_t* v_out;
    int64_t n_out, n_new;
    const int32_t* block_tables;
    int64_t bt_stride;
    const int32_t* context_lens;
    const int32_t* seq_lens_new;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t n_pages;
    int max_pages, page_size, row_chunks;
};

// grid = (row blocks, sequences): a workgroup widens kRowsPerBlock consecutive rows of one sequence.
constexpr int kRowsPerBlock = 32;

template <bool E2M1>
__global__ void __launch_bounds__(kThreads) mx_load_kernel(const MxLoadArgs a) {
    const int s = blockIdx.y;
    const int ctx = max(a.context_lens[s], 0), total = ctx + max(a.seq_lens_new[s], 0);
    const int row0 = blockIdx.x * kRowsPerBlock;
    if (row0 >= total) return;
    const int64_t out0 = a.cu_k[s], new0 = a.cu_q[s];
    const uint32_t row_chunks = a.row_chunks;
    const uint32_t n = min(kRowsPerBlock, total - row0) * row_chunks;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t rr = i / row_chunks, c = i - rr * row_chunks;
        const int r = row0 + static_cast<int>(rr);
        const int64_t dst = out0 + r;
        if (dst < 0 || dst >= a.n_out) continue;
        u32x4 kk, vv;
        if (r < ctx) {
            const int p = r / a.page_size;
            if (p >= a.max_pages) continue;
            const int64_t page = a.block_tables[s * a.bt_stride + p];
            if (page < 0 || page >= a.n_pages) continue;
            const int64_t chunk = (page * a.page_size + (r - p * a.page_size)) * row_chunks + c;
            const float ks = mx_scale_operand(a.k_scales[chunk >> 2]), vs = mx_scale_operand(a.v_scales[chunk >> 2]);
            if constexpr (E2M1) {
                kk = mx_widen8_e2m1(reinterpret_cast<const uint32_t*>(a.k_cache)[chunk], ks);
                vv = mx_widen8_e2m1(reinterpret_cast<const uint32_t*>(a.v_cache)[chunk], vs);
            } else {
                kk = mx_widen8_e4m3(reinterpret_cast<const u32x2*>(a.k_cache)[chunk], ks);
                vv = mx_widen8_e4m3(reinterpret_cast<const u32x2*>(a.v_cache)[chunk], vs);
            }
        } else {
            const int64_t t = new0 + (r - ctx);
            if (t < 0 || t >= a.n_new) continue;
            kk = *reinterpret_cast<const u32x4*>(a.k_new + t * a.k_new_stride + c * 8);
            vv = *reinterpret_cast<const u32x4*>(a.v_new + t * a.v_new_stride + c * 8);
        }
        __builtin_nontemporal_store(kk, reinterpret_cast<u32x4*>(a.k_out) + dst * row_chunks + c);
        __builtin_nontemporal_store(vv, reinterpret_cast<u32x4*>(a.v_out) + dst * row_chunks + c);
    }
}

bool is_mx(int kv_dtype) { return kv_dtype == DFX_KV_MX_E4M3 || kv_dtype == DFX_KV_MX_E2M1; }

}  // namespace
}  // namespace dfx

using namespace dfx;

extern "C" int dfx_kv_store_mx(const void* key, const void* value, int64_t key_stride, int64_t value_stride, void* k_cache,
                               void* v_cache, void* k_scales, void* v_scales, const void* slot_mapping, int slot_index_type,
                               int64_t n_tokens, int64_t n_slots, int n_kv_heads, int head_dim, int kv_dtype,
                               dfx_stream_t stream) {
    if (n_tokens < 0 || n_slots < 0 || n_kv_heads <= 0 || head_dim <= 0 || !is_mx(kv_dtype)) return DFX_ERR_INVALID_ARG;
    if (slot_index_type != DFX_INDEX_I32 && slot_index_type != DFX_INDEX_I64) return DFX_ERR_INVALID_ARG;
    if (head_dim % kMxBlock != 0) return DFX_ERR_UNSUPPORTED;
    if (n_tokens == 0) return DFX_OK;
    if (!key || !value || !k_cache || !v_cache || !k_scales || !v_scales || !slot_mapping) return DFX_ERR_INVALID_ARG;
    const int64_t row = static_cast<int64_t>(n_kv_heads) * head_dim;
    if (row > INT32_MAX || key_stride < row || value_stride < row) return DFX_ERR_INVALID_ARG;
    if (key_stride % 8 || value_stride % 8 || !aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache))
        return DFX_ERR_INVALID_ARG;
    MxStoreArgs a{};
    a.key = static_cast<const uint16_t*>(key);
    a.value = static_cast<const uint16_t*>(value);
    a.key_stride = key_stride;
    a.value_stride = value_stride;
    a.k_cache = static_cast<uint8_t*>(k_cache);
    a.v_cache = static_cast<uint8_t*>(v_cache);
    a.k_scales = static_cast<uint8_t*>(k_scales);
    a.v_scales = static_cast<uint8_t*>(v_scales);
    a.slots = slot_mapping;
    a.n_tokens = n_tokens;
    a.n_slots = n_slots;
    a.slot_type = slot_index_type;
    a.row_chunks = static_cast<int>(row / 8);
    const int64_t blocks = (n_tokens * a.row_chunks + kThreads - 1) / kThreads;
    if (blocks > UINT32_MAX / kThreads) return DFX_ERR_UNSUPPORTED;
    auto kern = kv_dtype == DFX_KV_MX_E2M1 ? mx_store_kernel<true> : mx_store_kernel<false>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    return launch_status();
}

extern "C" int dfx_kv_load_mx(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                              const void* k_new, const void* v_new, int64_t k_new_stride, int64_t v_new_stride, int64_t n_new,
                              void* k_out, void* v_out, int64_t n_out, const int32_t* block_tables, int64_t block_table_stride,
                              const int32_t* context_lens, const int32_t* seq_lens_new, const int32_t* cu_seqlens_q,
                              const int32_t* cu_seqlens_k, int num_seqs, int max_pages_per_seq, int64_t n_pages, int page_size,
                              int n_kv_heads, int head_dim, int64_t max_total_len, int kv_dtype, dfx_stream_t stream) {
    if (num_seqs < 0 || max_pages_per_seq < 0 || n_pages < 0 || page_size <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
        max_total_len < 0 || n_new < 0 || n_out < 0 || !is_mx(kv_dtype))
        return DFX_ERR_INVALID_ARG;
    if (head_dim % kMxBlock != 0 || num_seqs > 65535) return DFX_ERR_UNSUPPORTED;
    if (num_seqs == 0 || max_total_len == 0 || n_out == 0) return DFX_OK;
    if (!k_out || !v_out || !block_tables || !context_lens || !seq_lens_new || !cu_seqlens_q || !cu_seqlens_k)
        return DFX_ERR_INVALID_ARG;
    if (n_pages > 0 && (!k_cache || !v_cache || !k_scales || !v_scales)) return DFX_ERR_INVALID_ARG;
    if (n_new > 0 && (!k_new || !v_new)) return DFX_ERR_INVALID_ARG;
    const int64_t row = static_cast<int64_t>(n_kv_heads) * head_dim;
    if (row > INT32_MAX / kRowsPerBlock || (n_new > 0 && (k_new_stride < row || v_new_stride < row))) return DFX_ERR_INVALID_ARG;
    if (k_new_stride % 8 || v_new_stride % 8 || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_new) ||
        !aligned16(v_new) || !aligned16(k_out) || !aligned16(v_out))
        return DFX_ERR_INVALID_ARG;
    const int64_t row_blocks = (max_total_len + kRowsPerBlock - 1) / kRowsPerBlock;
    if (row_blocks > INT32_MAX / kThreads) return DFX_ERR_UNSUPPORTED;
    MxLoadArgs a{};
    a.k_cache = static_cast<const uint8_t*>(k_cache);
    a.v_cache = static_cast<const uint8_t*>(v_cache);
    a.k_scales = static_cast<const uint8_t*>(k_scales);
    a.v_scales = static_cast<const uint8_t*>(v_scales);
    a.k_new = static_cast<const uint16_t*>(k_new);
    a.v_new = static_cast<const uint16_t*>(v_new);
    a.k_new_stride = k_new_stride;
    a.v_new_stride = v_new_stride;
    a.k_out = static_cast<uint16_t*>(k_out);
    a.v_out = static_cast<uint16_t*>(v_out);
    a.n_out = n_out;
    a.n_new = n_new;
    a.block_tables = block_tables;
    a.bt_stride = block_table_stride;
    a.context_lens = context_lens;
    a.seq_lens_new = seq_lens_new;
    a.cu_q = cu_seqlens_q;
    a.cu_k = cu_seqlens_k;
    a.n_pages = n_pages;
    a.max_pages = max_pages_per_seq;
    a.page_size = page_size;
    a.row_chunks = static_cast<int>(row / 8);
    auto kern = kv_dtype == DFX_KV_MX_E2M1 ? mx_load_kernel<true> : mx_load_kernel<false>;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(row_blocks), static_cast<unsigned>(num_seqs)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    return launch_status();
}
