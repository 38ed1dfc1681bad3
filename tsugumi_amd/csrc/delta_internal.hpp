// delta_internal.hpp — what the gated delta rule's translation units share: the plan
// object, the kernels' arguments and the device's view of a batch.
#pragma once

#include "attn_internal.hpp"

struct tsg_delta {
    tsg_ctx* ctx = nullptr;
    int device = 0;  // the context's
    tsg_delta_config cfg{};
    uint32_t group = 0;       // value heads a key head serves
    uint32_t channels = 0;    // of the convolution
    uint32_t padded_key = 0;  // the kernels' key width: 64, 128 or 256
};

namespace tsg {

constexpr uint32_t kMaxDeltaKept = 8;  // rows a sequence in a decode call

// The sequences of a call, as the kernels see them.
struct DeltaSeqs {
    const uint32_t* row_starts;  // nullptr: uniform rows a sequence
    const uint32_t* in_slots;
    const uint32_t* out_slots;
    uint32_t* error;
    uint32_t num_seqs, rows, seq_rows, kept, num_slots;
};

struct DeltaArgs {
    DeltaSeqs seqs;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* a;
    const uint16_t* b;
    const float* a_log;
    const float* dt_bias;
    uint16_t* out;
    float* s;
    uint64_t slot_stride;
    uint32_t q_stride, k_stride, v_stride, a_stride, b_stride, out_stride;
    uint32_t value_heads, group, key_dim, value_dim;
    float scale, eps;
};

// Whether any row start falls or passes the rows: whose a row is, is unclear then.
__device__ __forceinline__ bool starts_wrong(const DeltaSeqs& d) {
    if (!d.row_starts) return false;
    const uint32_t lane = threadIdx.x & 63u;
    bool wrong = false;
    for (uint32_t s = lane; s < d.num_seqs; s += 64u) {
        const uint32_t lo = d.row_starts[s], hi = d.row_starts[s + 1u];
        wrong = wrong || lo > hi || hi > d.rows;
    }
    return __ballot(wrong) != 0;
}

struct DeltaSlot {
    uint32_t in;  // to read; 0 where it is past the pool
    bool fresh;   // no state before
    bool bad;     // past the pool
};
__device__ __forceinline__ DeltaSlot delta_slot(const DeltaSeqs& d, uint32_t s) {
    const uint32_t in = scalar_load(d.in_slots + s);
    const bool fresh = in == TSG_NO_SLOT, inside = in < d.num_slots;
    return DeltaSlot{inside ? in : 0u, fresh, !fresh && !inside};
}
struct DeltaSeq : DeltaSlot {
    uint32_t first, count;  // its rows
};
// Sequence s, where no row start is wrong.
__device__ __forceinline__ DeltaSeq delta_seq(const DeltaSeqs& d, uint32_t s) {
    DeltaSeq r{delta_slot(d, s), s * d.seq_rows, d.seq_rows};
    if (d.row_starts) {
        r.first = scalar_load(d.row_starts + s);
        r.count = scalar_load(d.row_starts + s + 1u) - r.first;
    }
    return r;
}

// Whether an out slot of sequence s is past the pool, or another sequence's in or
// out slot: the order of their reads and writes would be chance. Every kernel of
// a call comes to the same answer, and writes none of the sequence's states then.
// Every wave reads all sequences' slots, once, several loads in flight: quadratic in the
// sequences, and less than the states' way through memory up to some thousand of them (512
// sequences that keep 8 states of 4 heads of 64 x 64: 70 us; a pass over them for each state 176.
// 4096 that keep one 154 for 383).
template <uint32_t KEPT>
__device__ __forceinline__ bool out_slots_clash(const DeltaSeqs& d, uint32_t s) {
    const uint32_t lane = threadIdx.x & 63u, outs = d.num_seqs * d.kept, first = s * d.kept;
    uint32_t own[KEPT];
    uint32_t any = 0, clash = 0;
#pragma unroll
    for (uint32_t i = 0; i < KEPT; ++i) {
        own[i] = i < d.kept ? scalar_load(d.out_slots + first + i) : TSG_NO_SLOT;
        any |= own[i] != TSG_NO_SLOT;
        clash |= (own[i] != TSG_NO_SLOT) & (own[i] >= d.num_slots);
    }
    if (!any) return false;
    const auto mine = [&](uint32_t slot) {
        uint32_t hit = 0;
#pragma unroll
        for (uint32_t i = 0; i < KEPT; ++i) hit |= slot == own[i];
        return hit & (slot != TSG_NO_SLOT);
    };
#pragma unroll 4
    for (uint32_t t = lane; t < d.num_seqs; t += 64u) clash |= (t != s) & mine(d.in_slots[t]);
#pragma unroll 4
    for (uint32_t t = lane; t < outs; t += 64u)
        clash |= (t - first >= d.kept) & mine(d.out_slots[t]);
    return __ballot(clash) != 0;
}
__device__ __forceinline__ bool out_slots_clash(const DeltaSeqs& d, uint32_t s) {
    return d.kept == 1u ? out_slots_clash<1u>(d, s) : out_slots_clash<kMaxDeltaKept>(d, s);
}

// The rows in tiles of R: sequence s's begin at id starts[s] / R + s (a sequence
// without rows has one, of no rows); uniform ones at s * tiles a sequence. Uniform
// over the wave. kind 0: no tile; 1: rows first .. first + count - 1, `tile` of
// sequence `seq`; 2: wrong row starts (the tile's part of the rows as they lie).
struct DeltaTile {
    uint32_t kind, seq, tile, first, count;
};
template <uint32_t R>
__host__ __device__ __forceinline__ uint32_t delta_tiles(uint32_t rows, uint32_t num_seqs,
                                                         uint32_t seq_rows, bool ragged) {
    return ragged ? rows / R + num_seqs : num_seqs * ((seq_rows + R - 1u) / R);
}
template <uint32_t R>
__device__ __forceinline__ uint32_t delta_tile_base(const DeltaSeqs& d, const DeltaSeq& q,
                                                    uint32_t s) {
    return d.row_starts ? q.first / R + s : s * ((d.seq_rows + R - 1u) / R);
}
template <uint32_t R>
__device__ __forceinline__ DeltaTile delta_tile(const DeltaSeqs& d, uint32_t id) {
    DeltaTile r{1u, 0u, 0u, 0u, 0u};
    uint32_t first = 0, rows = d.seq_rows;
    if (!d.row_starts) {
        const uint32_t per = (d.seq_rows + R - 1u) / R;
        r.seq = id / per;
        r.tile = id % per;
        first = r.seq * d.seq_rows;
    } else {
        const uint32_t lane = threadIdx.x & 63u;
        uint32_t before = 0;  // sequences whose tiles begin at or before id
        bool wrong = false;
        for (uint32_t base = 0; base < d.num_seqs; base += 64u) {
            const uint32_t s = base + lane;
            const bool live = s < d.num_seqs;
            const uint32_t lo = live ? d.row_starts[s] : 0u, hi = live ? d.row_starts[s + 1u] : 0u;
            wrong = wrong || lo > hi || hi > d.rows;
            before += (uint32_t)__builtin_popcountll(__ballot(live && lo / R + s <= id));
        }
        if (__ballot(wrong)) {
            r.kind = 2u;
            r.first = id * R < d.rows ? id * R : d.rows;
            r.count = d.rows - r.first < R ? d.rows - r.first : R;
            return r;
        }
        if (before == 0u) return DeltaTile{0u, 0u, 0u, 0u, 0u};
        r.seq = before - 1u;
        first = scalar_load(d.row_starts + r.seq);
        rows = scalar_load(d.row_starts + r.seq + 1u) - first;
        r.tile = id - (first / R + r.seq);
    }
    if (r.tile * R >= rows && r.tile) return DeltaTile{0u, 0u, 0u, 0u, 0u};
    r.first = first + r.tile * R;
    r.count = rows - r.tile * R < R ? rows - r.tile * R : R;
    return r;
}

constexpr uint32_t kDeltaNan2 = 0x7E007E00u;  // two fp16 NaN
// delta_prefill.hip
tsg_status prepare_delta(const tsg_delta* delta);  // once a plan, its device current
uint64_t delta_scratch_bytes(const tsg_delta* delta, uint32_t rows, uint32_t num_seqs);
tsg_status launch_chunked(const tsg_delta* delta, const DeltaArgs& a, void* scratch,
                          tsg_stream stream);

}  // namespace tsg
