// attn_internal.hpp — what the attention's translation units share: the plan
// object, the kernels' arguments and the device's view of a batch.
#pragma once

#include "tsg_internal.hpp"

struct tsg_attn {
    tsg_ctx* ctx = nullptr;
    tsg_attn_config cfg{};
    uint32_t group = 0;       // query heads a key head serves
    uint32_t page_shift = 0;  // log2(page_tokens)
    uint32_t cell = 2;        // bytes of a cache element
};

namespace tsg {

// Bits of the context's error word (beside the kErr* of tsg_internal.hpp): a
// page id past the pool or a sequence longer than its page table (its rows
// are NaN, and nothing of them is appended); row starts that fall or pass the
// batch's rows.
constexpr uint32_t kErrAttnPage = 256u;
constexpr uint32_t kErrAttnLength = 512u;
constexpr uint32_t kErrAttnRows = 1024u;

constexpr uint32_t kMaxDecodeRows = 8;  // rows a sequence in a decode call (a speculative block)

struct AttnArgs {
    const uint16_t* q;
    uint16_t* out;
    const uint8_t* k;
    const uint8_t* v;
    const uint32_t* table;
    const uint32_t* lengths;
    const uint32_t* row_starts;  // nullptr: uniform rows a sequence
    uint32_t* error;
    uint64_t page_stride, head_stride;  // bytes
    uint32_t token_stride;              // bytes
    uint32_t q_stride, out_stride;      // elements
    uint32_t table_stride, num_seqs, rows, seq_rows, num_pages;
    uint32_t q_heads, kv_heads, group, dim, page_shift;
    uint32_t window, sinks;
    float scale_log2;  // logits to powers of two: scale * k_scale * log2(e)
    float v_scale;
};

struct SeqRows {
    uint32_t seq, first, count;  // its rows are first .. first + count - 1
    uint32_t length;             // tokens in the cache
    uint32_t bad;                // kErrAttnLength, kErrAttnRows or 0
};

// Rows and length of sequence s. Every value read from device memory is held
// to the batch's bounds before it is used.
__device__ __forceinline__ SeqRows seq_rows(const uint32_t* row_starts, const uint32_t* lengths,
                                            uint32_t s, uint32_t uniform, uint32_t rows,
                                            uint32_t capacity) {
    SeqRows r;
    r.seq = s;
    r.bad = 0u;
    if (row_starts) {
        const uint32_t lo = row_starts[s], hi = row_starts[s + 1];
        if (lo > hi || hi > rows) r.bad = kErrAttnRows;
        r.first = lo < rows ? lo : rows;
        const uint32_t end = hi < rows ? hi : rows;
        r.count = end > r.first ? end - r.first : 0u;
    } else {
        r.first = s * uniform;
        r.count = uniform;
    }
    const uint32_t n = lengths[s];
    if (n > capacity) r.bad = kErrAttnLength;
    r.length = n > capacity ? capacity : n;
    return r;
}

__device__ __forceinline__ void report(uint32_t* error, uint32_t bit) { atomicOr(error, bit); }

// The sequence that holds `row` (uniform over the wave), or num_seqs: with row
// starts the first s whose end lies past the row, 64 of them at a time. The
// waves of row 0 look at all of them and report starts that fall or pass the
// batch's rows.
__device__ __forceinline__ uint32_t find_seq(const uint32_t* row_starts, uint32_t num_seqs,
                                             uint32_t uniform, uint32_t rows, uint32_t row,
                                             uint32_t* error) {
    if (!row_starts) return row / uniform;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t found = num_seqs;
    for (uint32_t base = 0; base < num_seqs; base += 64u) {
        const uint32_t s = base + lane;
        const bool live = s < num_seqs;
        const uint32_t lo = live ? row_starts[s] : 0u, hi = live ? row_starts[s + 1u] : 0u;
        const uint64_t past = __ballot(live && hi > row);
        if (row == 0u && __ballot(lo > hi || hi > rows) && lane == 0) report(error, kErrAttnRows);
        if (past && found == num_seqs) {
            const int at = __builtin_ctzll(past);
            found = base + (uint32_t)at;
            if ((uint32_t)__builtin_amdgcn_readlane((int)lo, at) > row) return num_seqs;
            if (row != 0u) break;
        }
    }
    return found;
}

// Four e4m3 codes (one dword) as four fp16, exact.
__device__ __forceinline__ uint2 e4m3x4_to_f16(uint32_t w) {
    const h2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    const h2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Runs with the plan's device current; the caller's is restored on return.
struct DeviceScope {
    int before = -1;
    hipError_t status = hipSuccess;
    explicit DeviceScope(int device) {
        int now = 0;
        status = hipGetDevice(&now);
        if (status == hipSuccess && now != device) {
            status = hipSetDevice(device);
            if (status == hipSuccess) before = now;
        }
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// The argument checks every entry point makes, without a device (attn.hip).
tsg_status check_attn_config(const tsg_attn_config* c);
tsg_status check_attn_pages(const tsg_attn_config& c, const tsg_kv_pages* p);
tsg_status check_attn_batch(const tsg_attn_config& c, const tsg_attn_batch* b);
// Whether an attention call may start; fills its kernel's arguments.
tsg_status attn_args(const tsg_attn* attn, const tsg_kv_pages* pages, const tsg_attn_batch* batch,
                     const uint16_t* q, uint32_t q_stride, uint16_t* out, uint32_t out_stride,
                     AttnArgs* a);

}  // namespace tsg
