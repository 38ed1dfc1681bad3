// attn_decode.hip — attention of a few new rows of each sequence (1..8, or a
// prefill call's few rows of wide heads) over the paged cache.
//
// o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale q.k_j): every key and value is
// read once and used for the few rows of its head's group, so HBM bounds it
// (4 flop a byte and row) and, for short caches, the latency of the chain
// page table -> keys -> values -> join.
//
// A workgroup takes 16 rows (tokens x heads of one key head's group) and a run
// of key tiles; its four waves take the tiles in turn, 16 keys each, with no
// barrier between them: K and V go to the wave's own LDS (e4m3: K to the first
// operand's registers, V through registers), V to be read transposed, and the
// next tile's K is under way while this one's V is used. The waves' sums are
// joined in LDS; the workgroups of a split sequence leave partial sums in the plan's
// scratch, and the last of them to arrive adds those up in the order of the
// splits, so the result does not depend on which one it is.
//
// Measured on an MI355X: one sequence of 131,001 keys, 8 key heads of 128 (537
// MB) 116 us, 4.6 TB/s; 64 ragged sequences of up to 16,001 e4m3 keys (1.07 GB)
// 212 us, 5.0 TB/s (a large copy: 4.9); 1001 keys, 8 heads of 256: 10.6 us, of
// which the join takes 3.5 and the way to the first product 3.
#include "attn_internal.hpp"

namespace tsg {
namespace {

constexpr uint32_t kWaves = 4;
constexpr uint32_t kTile = 16;  // keys of a wave's tile; never more than a page

struct DecodeArgs {
    AttnArgs a;
    float* part_o;       // [slot][16][DP]
    float* part_ml;      // [slot][16][2]: reference m and sum
    uint32_t* arrivals;  // [slot]
    uint32_t chunks;     // runs of keys wanted, a head and row tile; 0: one a sequence
    uint32_t row_tiles;  // 16-row tiles of a sequence's rows and group
    uint32_t pairs;      // key heads * (most runs there can be)
    float join_cost;     // of a split in the join, against a tile's of its run
    PrefixArgs x;        // what the sequences share, summed up already
};

constexpr uint32_t kMinTiles = kWaves;  // key tiles worth a workgroup: one a wave
// Partial sums one workgroup joins: four heads over one key head of 128, 500,000
// keys 64 us (with up to 32 of them 167, 512 89), 131,000 35 (52, 41), but 32,000
// 23 (21, 23) and, eight of each over 8000 keys, 20 (13, 19).
constexpr uint32_t kMaxSplits = 128;
constexpr uint32_t kJoinLoads = 4;      // splits whose loads go out together
// Sequences of a batch with runs of one length. With one run each, 512 of 200 tokens
// (8 key heads of 128) take 83 us (balanced 102), 300 41 (48), 300 ragged ones of up to
// 4000 452 (470); but 300 with one of 100,000 among them 1237 (137). At 256, balanced,
// 39 and, with the long one, 128.
constexpr uint32_t kMaxBalanced = 256;

// The run of key tiles that workgroup `at` (of a head and row tile) takes. All
// runs of a batch have about the same length, whatever the sequences' lengths:
// the tiles of all sequences over the runs wanted.
struct Run {
    uint32_t seq, split, used, per;
    uint32_t slot;    // of the sequence's first partial sum
    uint32_t length;  // the sequence's
};
template <bool SHARED>
__device__ __forceinline__ uint32_t seq_key_tiles(const DecodeArgs& p, uint32_t s, uint32_t length) {
    const AttnArgs& a = p.a;
    if (length > (a.table_stride << a.page_shift)) return 0u;  // reported; its rows are NaN
    if constexpr (SHARED) {  // those behind the shared ones
        const uint32_t first = p.x.info[s].x / kTile, end = (length + kTile - 1u) / kTile;
        return end > first ? end - first : 0u;
    }
    const int32_t lo = (int32_t)length - (int32_t)a.seq_rows;
    return tile_span<kTile>(lo < 0 ? 0 : lo, (int32_t)length - 1, a.window, a.sinks).count;
}
template <bool SHARED>
__device__ __forceinline__ bool find_run(const DecodeArgs& p, uint32_t at, Run* r) {
    const AttnArgs& a = p.a;
    if (p.chunks == 0u) {
        if (at >= a.num_seqs) return false;
        *r = Run{at, 0u, 1u, 0xFFFFFFFFu, 0u, scalar_load(a.lengths + at)};
        return true;
    }
    const auto runs_of = [](uint32_t tiles, uint32_t per) {
        const uint32_t n = (tiles + per - 1u) / per;
        return n > 1u ? n : 1u;
    };
    // Of one sequence: a longer run takes longer, more runs are longer to join;
    // runs of r tiles and tiles / r splits cost the least together at r =
    // sqrt(tiles * join_cost). (4000 keys, 16 rows of 128: 30 us with 63 runs of
    // 4 tiles, 17 with longer ones; 32,000 keys 63 and 43.)
    const auto run_length = [&](uint32_t tiles, uint32_t per) {
        const uint32_t cap = (tiles + kMaxSplits - 1u) / kMaxSplits;
        const uint32_t even = (uint32_t)__builtin_sqrtf((float)tiles * p.join_cost) + 1u;
        const uint32_t least = cap > even ? cap : even;
        return per > least ? per : least;
    };
    if (a.num_seqs == 1u) {
        const uint32_t length = scalar_load(a.lengths);
        const uint32_t tiles = seq_key_tiles<SHARED>(p, 0u, length);
        const uint32_t even = (tiles + p.chunks - 1u) / p.chunks;
        const uint32_t per = run_length(tiles, even > kMinTiles ? even : kMinTiles);
        *r = Run{0u, at, runs_of(tiles, per), per, 0u, length};
        return at < r->used;
    }
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t first = 0;  // the first 64 lengths are read once
    uint64_t total = 0;  // of 256 sequences of up to 2^26 tiles each
    for (uint32_t base = 0; base < a.num_seqs; base += 64u) {
        const uint32_t length = base + lane < a.num_seqs ? a.lengths[base + lane] : 0u;
        uint32_t n = base + lane < a.num_seqs ? seq_key_tiles<SHARED>(p, base + lane, length) : 0u;
        if (base == 0u) first = length;
        n -= n >> 26;  // 64 of them stay under 2^32
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += (uint32_t)__shfl_xor((int)n, o, 64);
        total += (uint32_t)__builtin_amdgcn_readfirstlane((int)n);
    }
    // at least total / chunks: no more runs then than chunks + sequences (the grid), and
    // fewer than 2 chunks of split sequences (the scratch)
    uint32_t per = total >> 31 ? ((uint32_t)(total >> 8) / p.chunks + 1u) << 8
                               : ((uint32_t)total + p.chunks - 1u) / p.chunks;
    per = per > kMinTiles ? per : kMinTiles;
    uint32_t slots = 0;
    for (uint32_t base = 0; base < a.num_seqs; base += 64u) {
        const bool live = base + lane < a.num_seqs;
        const uint32_t length = base == 0u ? first : live ? a.lengths[base + lane] : 0u;
        const uint32_t tiles = live ? seq_key_tiles<SHARED>(p, base + lane, length) : 0u;
        const uint32_t own = run_length(tiles, per);
        const uint32_t runs = live ? runs_of(tiles, own) : 0u;
        // runs, and above them those of split sequences: both sums stay under 2^16
        const uint32_t both = runs | (runs > 1u ? runs << 16 : 0u);
        uint32_t sum = both;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = (uint32_t)__shfl_up((int)sum, (unsigned)o, 64);
            if (lane >= (uint32_t)o) sum += v;
        }
        const uint64_t past = __ballot((sum & 0xFFFFu) > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            const uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)(sum - both), l);
            r->seq = base + (uint32_t)l;
            r->split = at - (before & 0xFFFFu);
            r->used = (uint32_t)__builtin_amdgcn_readlane((int)runs, l);
            r->per = (uint32_t)__builtin_amdgcn_readlane((int)own, l);
            r->slot = slots + (before >> 16);
            r->length = (uint32_t)__builtin_amdgcn_readlane((int)length, l);
            return true;
        }
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        at -= all & 0xFFFFu;
        slots += all >> 16;
    }
    return false;
}

// Wide heads' query fragments, the same for the four waves, are read from LDS
// for each tile: in registers (16 x DP fp16, DP / 8 of them) they would spill.
template <int DP>
constexpr bool kQueryInLds = DP >= 256;

template <int DP>
constexpr uint32_t kMarkBytes = kWaves * 16u * DP / 4u;

template <int DP>
constexpr uint32_t decode_lds_bytes() {
    // the waves' K and V tiles, and in their place at the end the waves' sums
    return kWaves * 16u * (DP + 4u) * 4u + 2u * kWaves * 16u * 4u + 32u +
           (kQueryInLds<DP> ? 16u * DP * 2u : 0u) + kMarkBytes<DP>;
}

// Place of the 32-byte pieces of key t's row in the wave's V tile: piece b lies
// at b ^ value_swizzle(t), so that the eight keys that half a wave reads at
// once (transposing) lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t value_swizzle(uint32_t t) {
    return DP >= 128 ? t & 7u : (t >> 1) & 3u;
}

template <int DP>
__device__ __forceinline__ uint32_t key_swizzle(uint32_t t) {  // of 16-byte chunks of K
    return DP >= 128 ? t & 15u : (t >> 1) & 7u;
}

// fp16 rows go straight from memory to LDS, K as well; e4m3 codes (and rows of
// other widths, whose ends are zeros) pass through registers.
template <bool E4M3, bool FULL>
constexpr bool kDirect = !E4M3 && FULL;
// Waves a SIMD's registers are shared by.
template <int DP, bool E4M3, bool FULL>
constexpr int kSimdWaves = kDirect<E4M3, FULL> ? (DP <= 128 ? 4 : 2)
                                               : (DP <= 128 ? 3 : DP <= 256 ? 2 : 1);

// SHARED: the keys behind those that a group of sequences shares, whose sums are there.
template <int DP, bool E4M3, bool FULL, bool SHARED = false>
__global__ __launch_bounds__(256, (kSimdWaves<DP, E4M3, FULL>)) void decode_kernel(DecodeArgs p) {
    constexpr uint32_t NS = DP / 32, NB = DP / 16;   // key-product steps, value blocks
    constexpr uint32_t CELL = E4M3 ? 1 : 2;
    constexpr uint32_t KL = E4M3 ? NS / 2 : NS;      // 16-byte K loads of a lane
    constexpr uint32_t CPR = DP * CELL / 16;         // 16-byte chunks of a cache row
    constexpr uint32_t TPI = 64 / CPR;               // keys one V load instruction covers
    constexpr uint32_t VL = kTile / TPI;             // V loads of a lane
    constexpr bool DMA = kDirect<E4M3, FULL>;
    extern __shared__ __align__(16) uint8_t smem[];
    const AttnArgs& a = p.a;

    uint32_t pair = blockIdx.x, rt = 0;
    if (p.row_tiles > 1u) {  // the row tiles of a pair share its keys: one XCD
        const uint32_t j = blockIdx.x >> 3;
        rt = j % p.row_tiles;
        pair = (j / p.row_tiles) * 8u + (blockIdx.x & 7u);
        if (pair >= p.pairs) return;
    }
    const uint32_t kvh = pair % a.kv_heads;
    Run run;
    if (!find_run<SHARED>(p, pair / a.kv_heads, &run)) return;
    const uint32_t s = run.seq;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t i16 = lane & 15u, g = lane >> 4;
    const uint32_t capacity = a.table_stride << a.page_shift;
    const uint32_t bad_length = run.length > capacity ? kErrAttnLength : 0u;
    const SeqRows sr{s, s * a.seq_rows, a.seq_rows, bad_length ? capacity : run.length, bad_length};

    const uint32_t rows = sr.count * a.group, r0 = rt * kDecodeTileRows;
    const uint32_t last = r0 + 15u < rows ? r0 + 15u : rows - 1u;
    const int32_t base = (int32_t)sr.length - (int32_t)sr.count;
    // positions of all of the sequence's rows: its row tiles take the same runs
    const int32_t p_lo = base, p_hi = (int32_t)sr.length - 1;
    TileSpan span = tile_span<kTile>(p_lo < 0 ? 0 : p_lo, p_hi, a.window, a.sinks);
    uint32_t shared = 0, shared_splits = 1;  // tokens
    bool bad_groups = false;
    if constexpr (SHARED) {
        shared = scalar_load(&p.x.info[s].x);
        const uint32_t y = scalar_load(&p.x.info[s].y);
        bad_groups = (y & 1u) != 0u;
        shared_splits = y >> 1;
        span.first = shared / kTile;
        span.count = span.count > span.first ? span.count - span.first : 0u;
    }
    const uint32_t used = run.used;
    const uint32_t tile_first = run.split * run.per;  // one run: split 0
    const uint32_t tile_end =
        used > 1u && tile_first + run.per < span.count ? tile_first + run.per : span.count;

    // the lane's query row as the second operand of K Q^T; step s of the
    // product takes, from lane group g, head elements qdim(s) ..
    const auto qdim = [&](uint32_t st) {
        return E4M3 ? 64u * (st >> 1) + 16u * g + 8u * (st & 1u) : 32u * st + 8u * g;
    };
    const uint32_t row = r0 + i16 < rows ? r0 + i16 : last;
    const uint32_t tok = row / a.group;
    const int32_t pos = base + (int32_t)tok;
    const uint16_t* q = a.q + (uint64_t)(sr.first + tok) * a.q_stride +
                        (uint64_t)(kvh * a.group + row % a.group) * a.dim;
    const auto load_q = [&](uint32_t st) -> h8_t {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (FULL || qdim(st) < a.dim) u = load_query(q + qdim(st), a.q_sign);
        return __builtin_bit_cast(h8_t, u);
    };
    constexpr bool QL = kQueryInLds<DP>;
    h8_t* qs = reinterpret_cast<h8_t*>(smem + decode_lds_bytes<DP>() - kMarkBytes<DP> - 16u * DP * 2u) + lane;
    h8_t qf[QL ? NS / kWaves : NS];  // QL: the steps that this wave stages
#pragma unroll
    for (uint32_t st = 0; st < (QL ? NS / kWaves : NS); ++st)
        qf[st] = load_q(QL ? wave * (NS / kWaves) + st : st);

    const uint32_t* table = a.table + (uint64_t)s * a.table_stride;
    const uint32_t page_mask = (1u << a.page_shift) - 1u;
    const uint64_t head_off = (uint64_t)kvh * a.head_stride;
    bool bad = false;
    // byte offset of a tile's first key in the pools
    const auto tile_offset = [&](uint32_t idx) -> uint64_t {
        const uint32_t t = span.key_tile(idx) * kTile;
        uint32_t page = scalar_load(table + (t >> a.page_shift));
        if (page >= a.num_pages) {
            bad = true;
            page = 0u;
        }
        return page * a.page_stride + head_off + (uint64_t)(t & page_mask) * a.token_stride;
    };

    const uint32_t k_lane = i16 * a.token_stride;  // lane i16 of each group holds key i16
    const uint32_t v_chunk = lane % CPR;
    const bool v_in = FULL || v_chunk * 16u < a.dim * CELL;
    const uint32_t v_lane = (lane / CPR) * a.token_stride + (v_in ? v_chunk * 16u : 0u);
    uint8_t* vs = smem + wave * (kTile * DP * 2u * (DMA ? 2u : 1u));
    uint8_t* ks = vs + kTile * DP * 2u;  // DMA only
    const uint32_t v_tok = lane / CPR, v_row = v_tok * a.token_stride;
    const uint32_t vs_lds = (uint32_t)(uintptr_t)vs, ks_lds = (uint32_t)(uintptr_t)ks;
    uint4 kreg[DMA ? 1 : KL], vreg[DMA ? 1 : VL];
    const auto load_k = [&](uint64_t off) {
        if constexpr (DMA) {
            // offsets are formed here each time (opaque lane): hoisted they would be
            // spilled, and a reload's wait would drain the loads under way
            uint32_t c = v_chunk;
            asm("" : "+v"(c));
#pragma unroll
            for (uint32_t n = 0; n < VL; ++n)
                dma16(a.k + (off + n * TPI * a.token_stride),
                      v_row + 16u * (c ^ key_swizzle<DP>(n * TPI + v_tok)), ks_lds + n * 1024u);
            return;
        }
        const uint8_t* kp = a.k + off;
#pragma unroll
        for (uint32_t l = 0; l < KL; ++l) {
            const uint32_t byte = 64u * l + 16u * g;
            const bool in = FULL || byte < a.dim * CELL;
            const uint4 x = load16_nt(kp + (k_lane + (in ? byte : 0u)));
            kreg[l] = in ? x : make_uint4(0, 0, 0, 0);
        }
    };
    const auto load_v = [&](uint64_t off) {
        if constexpr (DMA) {
            uint32_t c = v_chunk;
            asm("" : "+v"(c));
#pragma unroll
            for (uint32_t n = 0; n < VL; ++n)
                dma16(a.v + (off + n * TPI * a.token_stride),
                      v_row + 16u * (c ^ (2u * value_swizzle<DP>(n * TPI + v_tok))),
                      vs_lds + n * 1024u);
            return;
        }
#pragma unroll
        for (uint32_t n = 0; n < VL; ++n)
            vreg[n] = load16_nt(a.v + (off + n * TPI * a.token_stride) + v_lane);
    };
    const auto k_frag = [&](uint32_t st) -> h8_t {
        if constexpr (E4M3) {
            const uint4 w = kreg[st >> 1];
            const uint2 lo = e4m3x4_to_f16(st & 1u ? w.z : w.x), hi = e4m3x4_to_f16(st & 1u ? w.w : w.y);
            return __builtin_bit_cast(h8_t, make_uint4(lo.x, lo.y, hi.x, hi.y));
        } else if constexpr (DMA) {
            return *reinterpret_cast<const h8_t*>(
                ks + i16 * (DP * 2u) + 16u * ((4u * st + g) ^ key_swizzle<DP>(i16)));
        } else {
            return __builtin_bit_cast(h8_t, kreg[st]);
        }
    };

    const uint32_t tr_tok = 4u * g + (i16 >> 2);  // accumulator register j of group g is key 4 g + j
    const uint32_t tr_base =
        tr_tok * (DP * 2u) + 8u * (i16 & 3u) + 32u * value_swizzle<DP>(tr_tok);
    const auto v_frag = [&](uint32_t b) -> h4_t {
        return __builtin_bit_cast(h4_t, lds_read_tr(vs + (tr_base ^ (32u * b))));
    };

    // The product would make NaN of the weight 0 of a row that does not see an
    // infinity's or NaN's key: they are taken out of the V tile and noted in
    // `marks` (two bits, +inf and -inf, NaN both, for each element of the rows
    // that see the key), which go onto the sums at the end.
    uint32_t* marks =
        reinterpret_cast<uint32_t*>(smem + decode_lds_bytes<DP>() - kMarkBytes<DP>) +
        wave * (kMarkBytes<DP> / 4u / kWaves);  // [row][DP / 16]
    bool marked = false;
    const auto take_out = [&](uint32_t t0) {
        if (!marked)
            for (uint32_t n = lane; n < DP; n += 64u) marks[n] = 0u;
        marked = true;
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (uint32_t n = lane; n < kTile * DP; n += 64u) {
            uint16_t* v = reinterpret_cast<uint16_t*>(vs) + n;
            const uint32_t bits = *v;
            if ((bits & 0x7C00u) != 0x7C00u) continue;
            *v = 0;
            const uint32_t t = n / DP, e = n % DP;
            const uint32_t dim = 8u * ((e / 8u) ^ (2u * value_swizzle<DP>(t))) + e % 8u;
            const uint32_t mark = (bits & 0x3FFu ? 3u : bits & 0x8000u ? 2u : 1u) << (2u * (dim & 15u));
#pragma unroll 1
            for (uint32_t r = 0; r <= last - r0; ++r)
                if (key_seen((int32_t)(t0 + t), base + (int32_t)((r0 + r) / a.group), a.window,
                             a.sinks))
                    atomicOr(marks + r * (DP / 16u) + dim / 16u, mark);
        }
        __builtin_amdgcn_wave_barrier();
    };

    f4_t o[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) o[b] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNoKey, l = 0.0f;

    uint32_t idx = tile_first + wave;
    if (sr.bad) idx = tile_end;
    uint64_t off = 0;
    if (idx < tile_end) {
        off = tile_offset(idx);
        load_k(off);
        load_v(off);
    }
    if constexpr (QL) {
#pragma unroll
        for (uint32_t st = 0; st < NS / kWaves; ++st)
            qs[(wave * (NS / kWaves) + st) * 64u] = qf[st];
        lds_barrier();
    }
    for (; idx < tile_end; idx += kWaves) {
        const uint32_t t0 = span.key_tile(idx) * kTile;
        const bool whole = tile_seen_whole<kTile>(t0, p_lo, p_hi, a.window, a.sinks);
        if constexpr (DMA) wait_loads<VL>();  // K is there, V still on its way
        f4_t sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t st = 0; st < NS; ++st) {
            const h8_t qx = QL ? qs[st * 64u] : qf[QL ? 0 : st];
            sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k_frag(st), qx, sc, 0, 0, 0);
            if (QL && st % 4u == 3u) __builtin_amdgcn_sched_barrier(0);  // few reads ahead: registers
        }
        const bool more = idx + kWaves < tile_end;
        if (more) {
            off = tile_offset(idx + kWaves);
            if constexpr (DMA) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K was read
            load_k(off);
        }
        // Keys that no row sees (behind the last, before the window) may hold
        // anything: their V becomes zeros.
        bool tainted = false;  // an infinity or NaN that some row sees and some may not
        uint32_t seen = 0xFu;
        if (!whole) {
            if constexpr (DMA) wait_loads<0>();
            uint32_t found = 0;
#pragma unroll
            for (uint32_t n = 0; n < VL; ++n) {
                uint4* at = reinterpret_cast<uint4*>(vs) + n * 64u + lane;
                uint4 x = DMA ? *at : vreg[DMA ? 0 : n];
                const uint32_t keep =
                    keys_seen<1>(t0 + n * TPI + v_tok, p_lo, p_hi, a.window, a.sinks) ? ~0u : 0u;
                x = make_uint4(x.x & keep, x.y & keep, x.z & keep, x.w & keep);
                if constexpr (DMA) *at = x;
                else vreg[n] = x;
                found |= not_finite<E4M3>(x.x) | not_finite<E4M3>(x.y) | not_finite<E4M3>(x.z) |
                         not_finite<E4M3>(x.w);
            }
            tainted = __ballot(found != 0u) != 0;
            seen = 0u;
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e)
                seen |= (uint32_t)key_seen((int32_t)(t0 + 4u * g + e), pos, a.window, a.sinks) << e;
        }
        // V into the wave's LDS
#pragma unroll
        for (uint32_t n = 0; n < (DMA ? 0u : VL); ++n) {
            const uint32_t t = n * TPI + v_tok;
            if constexpr (E4M3) {
                const uint2 x0 = e4m3x4_to_f16(vreg[n].x), x1 = e4m3x4_to_f16(vreg[n].y);
                const uint2 x2 = e4m3x4_to_f16(vreg[n].z), x3 = e4m3x4_to_f16(vreg[n].w);
                uint4* dst = reinterpret_cast<uint4*>(
                    vs + t * (DP * 2u) + 32u * (v_chunk ^ value_swizzle<DP>(t)));
                dst[0] = make_uint4(x0.x, x0.y, x1.x, x1.y);
                dst[1] = make_uint4(x2.x, x2.y, x3.x, x3.y);
            } else {
                *reinterpret_cast<uint4*>(vs + t * (DP * 2u) +
                                          16u * (v_chunk ^ (2u * value_swizzle<DP>(t)))) = vreg[n];
            }
        }
        if (!DMA && more) load_v(off);

        float x[4];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e)
            x[e] = (seen >> e) & 1u ? sc[e] : -__builtin_inff();
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (__ballot((top - m) * a.scale_log2 > kMaxLag)) {
            const float mn = fmaxf(m, max_across32(max_across16(top)));
            const float alpha = __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
            m = mn;
            l *= alpha;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) o[b] *= alpha;
        }
        h4_t w;
#pragma unroll
        for (uint32_t e = 0; e < 4u; e += 2u) {
            const h2_t two = weight_pair(__builtin_fmaf(x[e] - m, a.scale_log2, kWeightBias),
                                         __builtin_fmaf(x[e + 1] - m, a.scale_log2, kWeightBias));
            l = dot2(two, h2_t{1, 1}, l);
            w[e] = two[0];
            w[e + 1] = two[1];
        }
        if constexpr (DMA) {  // V is there, the next K still on its way
            if (more) wait_loads<VL>();
            else wait_loads<0>();
        }
        __builtin_amdgcn_wave_barrier();  // the wave's own LDS: its operations stay in order
        if (tainted) take_out(t0);
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            o[b] = __builtin_amdgcn_mfma_f32_16x16x16f16(v_frag(b), w, o[b], 0, 0, 0);
            if (QL && b % 8u == 7u) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_wave_barrier();
        if constexpr (DMA) {
            if (more) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V was read
                load_v(off);
            }
        }
    }
    l = sum_across32(sum_across16(l));
    if (bad || sr.bad) {
        l = __builtin_nanf("");
        if (lane == 0) report(a.error, sr.bad ? sr.bad : kErrAttnPage);
    }
    if (SHARED && bad_groups) l = __builtin_nanf("");  // reported

    // the four waves' sums: lane (row i16, g) holds elements 16 b + 4 g .. + 3
    float* so = reinterpret_cast<float*>(smem);
    float* sm = so + kWaves * 16u * (DP + 4u);
    float* sl = sm + kWaves * 16u;
    uint32_t* sx = reinterpret_cast<uint32_t*>(sl + kWaves * 16u);  // which waves have marks
    uint32_t* flag = sx + kWaves;
    __syncthreads();  // every wave is done with its V
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
        *reinterpret_cast<f4_t*>(so + (wave * 16u + i16) * (DP + 4u) + 16u * b + 4u * g) = o[b];
    if (g == 0) {
        sm[wave * 16u + i16] = m;
        sl[wave * 16u + i16] = l;
    }
    if (lane == 0) sx[wave] = marked ? 1u : 0u;
    __syncthreads();

    constexpr uint32_t C8 = DP / 8;                      // 8-element pieces of a row
    constexpr uint32_t PIECES = (16u * C8 + 255u) / 256u;  // of a thread
    const uint32_t live = last - r0 + 1u;
    const auto slot_of = [&](uint32_t split) {  // its place among the partial sums
        return ((uint64_t)(run.slot + split) * a.kv_heads + kvh) * p.row_tiles + rt;
    };
    const auto out_at = [&](uint32_t r, uint32_t c) {
        const uint32_t t = (r0 + r) / a.group;
        return a.out + (uint64_t)(sr.first + t) * a.out_stride +
               (uint64_t)(kvh * a.group + (r0 + r - t * a.group)) * a.dim + 8u * c;
    };
    const auto emit = [&](uint32_t r, uint32_t c, const float* acc, float sum) {
        uint16_t* out = out_at(r, c);
        const float inv = row_inverse(sum, base + (int32_t)((r0 + r) / a.group), a.v_scale);
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            h[e] = (uint32_t)f32_to_f16(acc[2 * e] * inv) |
                   ((uint32_t)f32_to_f16(acc[2 * e + 1] * inv) << 16);
        *reinterpret_cast<uint4*>(out) = make_uint4(h[0], h[1], h[2], h[3]);
    };
    // The sums of the shared keys, every ways-th split of them, added to a row's piece.
    const auto add_shared = [&](uint32_t r, uint32_t c, float* acc, float& sum, float& mm,
                                uint32_t way, uint32_t ways) {
        const uint32_t splits = prefix_split(p.x, shared_splits, shared / kTileKeys<DP>).used;
        const uint64_t first = (uint64_t)kvh * p.x.splits * p.x.rows + s * rows + r0 + r;
#pragma unroll 1
        for (uint32_t w0 = way; w0 < splits; w0 += kJoinLoads * ways) {
            f4_t lo[kJoinLoads], hi[kJoinLoads];
            float2 ml[kJoinLoads];
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) {
                const uint32_t w = w0 + k * ways < splits ? w0 + k * ways : w0;
                const uint64_t at = first + (uint64_t)w * p.x.rows;
                ml[k] = *reinterpret_cast<const float2*>(p.x.part_ml + at * 2u);
                const f4_t* src = reinterpret_cast<const f4_t*>(p.x.part_o + at * DP + 8u * c);
                lo[k] = src[0];
                hi[k] = src[1];
            }
            float mn = mm;
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) mn = fmaxf(mn, ml[k].x);
            const float f0 = __builtin_amdgcn_exp2f((mm - mn) * a.scale_log2);
            mm = mn;
            sum *= f0;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= f0;
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) {
                if (w0 + k * ways >= splits) continue;
                const float f = __builtin_amdgcn_exp2f((ml[k].x - mn) * a.scale_log2);
                sum += ml[k].y * f;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += (e < 4 ? lo[k][e & 3] : hi[k][e & 3]) * f;
            }
        }
    };
    // neighbouring lanes that share a piece, where the row's keys are this workgroup's and
    // shared ones: the first has the former, each some splits of the latter
    uint32_t share_log2 = 0;
    if constexpr (SHARED)
        if (used == 1u && shared)
            while ((live * C8 << (share_log2 + 1u)) <= 256u && share_log2 < 5u) ++share_log2;
    const uint32_t share_way = threadIdx.x & ((1u << share_log2) - 1u);
#pragma unroll 1
    for (uint32_t n = 0; n < PIECES; ++n) {
        const uint32_t piece = (threadIdx.x >> share_log2) + 256u * n, r = piece / C8, c = piece % C8;
        if (r >= live || 8u * c >= a.dim) continue;
        float mm = sm[r];
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) mm = fmaxf(mm, sm[w * 16u + r]);
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            if (SHARED && share_way) break;
            const float f = __builtin_amdgcn_exp2f((sm[w * 16u + r] - mm) * a.scale_log2);
            sum += sl[w * 16u + r] * f;
            const float* src = so + (w * 16u + r) * (DP + 4u) + 8u * c;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += src[e] * f;
        }
        for (uint32_t w = 0; w < kWaves; ++w) {
            if (!sx[w] || (SHARED && share_way)) continue;
            const uint32_t mark = reinterpret_cast<const uint16_t*>(
                smem + decode_lds_bytes<DP>() - kMarkBytes<DP>)[(w * 16u + r) * (DP / 8u) + c];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (mark >> (2 * e) & 1u) acc[e] += __builtin_inff();
                if (mark >> (2 * e) & 2u) acc[e] -= __builtin_inff();
            }
        }
        if (used == 1u) {
            if constexpr (SHARED) {
                add_shared(r, c, acc, sum, mm, share_way, 1u << share_log2);
                // the lanes of a piece are all here
                for (uint32_t o = 1; o < 1u << share_log2; o <<= 1) {
                    const float m2 = __shfl_xor(mm, (int)o, 64), mn = fmaxf(mm, m2);
                    const float f0 = __builtin_amdgcn_exp2f((mm - mn) * a.scale_log2);
                    const float f1 = __builtin_amdgcn_exp2f((m2 - mn) * a.scale_log2);
                    mm = mn;
                    sum = sum * f0 + __shfl_xor(sum, (int)o, 64) * f1;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc[e] = acc[e] * f0 + __shfl_xor(acc[e], (int)o, 64) * f1;
                }
                if (share_way) continue;
            }
            emit(r, c, acc, sum);
        } else {
            const uint64_t slot = slot_of(run.split) * 16u + r;
            float* dst = p.part_o + slot * DP + 8u * c;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t two = (uint64_t)__float_as_uint(acc[2 * e]) |
                                     ((uint64_t)__float_as_uint(acc[2 * e + 1]) << 32);
                st_coherent(reinterpret_cast<uint64_t*>(dst) + e, two);
            }
            if (c == 0)
                st_coherent(reinterpret_cast<uint64_t*>(p.part_ml) + slot,
                            (uint64_t)__float_as_uint(mm) | ((uint64_t)__float_as_uint(sum) << 32));
        }
    }
    if (used == 1u) return;

    // The last workgroup of the sequence, head and row tile to arrive joins the
    // splits: `ways` neighbouring lanes share an 8-element piece, each adds up
    // every ways-th split, in order, four at a time from loads that go out
    // together; then the lanes' sums are added in a fixed order.
    const uint32_t pieces = live * C8;
    uint32_t ways_log2 = 0;  // at most 5: a row has at least eight pieces
    while ((pieces << (ways_log2 + 1u)) <= 256u && (2u << ways_log2) <= used) ++ways_log2;
    const uint32_t ways = 1u << ways_log2, way = threadIdx.x & (ways - 1u);
    const uint32_t slot0 = (uint32_t)slot_of(0);
    wait_vector_memory();
    lds_barrier();
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(p.arrivals + slot0, 1u, __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT);
        *flag = before == used - 1u ? 1u : 0u;
    }
    lds_barrier();
    if (!*flag) return;
    const uint32_t step = a.kv_heads * p.row_tiles * 16u;
#pragma unroll 1
    for (uint32_t n = 0; n < pieces; n += 256u >> ways_log2) {
        const uint32_t piece = n + (threadIdx.x >> ways_log2), r = piece / C8, c = piece % C8;
        const bool in = piece < pieces && 8u * c < a.dim;
        float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f, mm = kNoKey;
        uint32_t at = slot0 * 16u + (in ? r : 0u) + way * step;  // the scratch is under 4 GiB
#pragma unroll 1
        for (uint32_t w0 = way; w0 < used; w0 += kJoinLoads * ways, at += kJoinLoads * ways * step) {
            uint4 lo[kJoinLoads], hi[kJoinLoads];
            uint64_t ml[kJoinLoads];
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) {
                const uint32_t at_k = w0 + k * ways < used ? at + k * ways * step : at;
                const uint32_t byte = (at_k * (uint32_t)DP + 8u * c) * 4u;
                ml[k] = ld_coherent(reinterpret_cast<const uint64_t*>(
                    reinterpret_cast<const uint8_t*>(p.part_ml) + at_k * 8u));
                lo[k] = ld_coherent16(reinterpret_cast<const uint8_t*>(p.part_o) + byte);
                hi[k] = ld_coherent16(reinterpret_cast<const uint8_t*>(p.part_o) + byte + 16u);
            }
            float mk[kJoinLoads], mn = mm;
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) {
                mk[k] = __uint_as_float((uint32_t)ml[k]);
                mn = fmaxf(mn, mk[k]);
            }
            const float f0 = __builtin_amdgcn_exp2f((mm - mn) * a.scale_log2);
            mm = mn;
            sum *= f0;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= f0;
#pragma unroll
            for (uint32_t k = 0; k < kJoinLoads; ++k) {
                const bool have = w0 + k * ways < used;
                const float f = have ? __builtin_amdgcn_exp2f((mk[k] - mn) * a.scale_log2) : 0.0f;
                const uint32_t u[8] = {lo[k].x, lo[k].y, lo[k].z, lo[k].w,
                                       hi[k].x, hi[k].y, hi[k].z, hi[k].w};
                if (have) {
                    sum += __uint_as_float((uint32_t)(ml[k] >> 32)) * f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] += __uint_as_float(u[e]) * f;
                }
            }
        }
        if constexpr (SHARED)
            if (in) add_shared(r, c, acc, sum, mm, way, ways);
        for (uint32_t o = 1; o < ways; o <<= 1) {
            const float m2 = __shfl_xor(mm, (int)o, 64), mn = fmaxf(mm, m2);
            const float f0 = __builtin_amdgcn_exp2f((mm - mn) * a.scale_log2);
            const float f1 = __builtin_amdgcn_exp2f((m2 - mn) * a.scale_log2);
            mm = mn;
            sum = sum * f0 + __shfl_xor(sum, (int)o, 64) * f1;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f0 + __shfl_xor(acc[e], (int)o, 64) * f1;
        }
        if (in && way == 0u) emit(r, c, acc, sum);
    }
    if (threadIdx.x == 0) st_coherent(p.arrivals + slot0, 0u);  // for the next call
}

typedef void (*DecodeKernel)(DecodeArgs);

template <int DP, bool SHARED>
DecodeKernel kernel_of(bool e4m3, bool full) {
    if (e4m3)
        return full ? decode_kernel<DP, true, true, SHARED> : decode_kernel<DP, true, false, SHARED>;
    return full ? decode_kernel<DP, false, true, SHARED> : decode_kernel<DP, false, false, SHARED>;
}

struct Variant {
    DecodeKernel kernel, shared;
    uint32_t lds;
};
template <int DP>
Variant variant(bool e4m3, bool full) {
    return {kernel_of<DP, false>(e4m3, full), kernel_of<DP, true>(e4m3, full), decode_lds_bytes<DP>()};
}
Variant variant_of(const tsg_attn* attn) {
    const bool e4m3 = attn->cfg.kv_type == TSG_KV_E4M3;
    const bool full = attn->cfg.head_dim == attn->padded_dim;
    switch (attn->padded_dim) {
        case 64: return variant<64>(e4m3, full);
        case 128: return variant<128>(e4m3, full);
        case 256: return variant<256>(e4m3, full);
        default: return variant<512>(e4m3, full);
    }
}

}  // namespace

tsg_status prepare_decode(const tsg_attn* attn) {
    const Variant v = variant_of(attn);
    for (DecodeKernel kernel : {v.kernel, v.shared})
        TSG_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)v.lds));
    return TSG_OK;
}

tsg_status launch_decode(const tsg_attn* attn, const AttnArgs& a, tsg_stream stream,
                         const PrefixArgs* prefix) {
    DecodeArgs p{};
    p.a = a;
    if (prefix) p.x = *prefix;
    p.row_tiles = (a.seq_rows * a.group + kDecodeTileRows - 1u) / kDecodeTileRows;
    // As many runs as workgroups fit the card at once (LDS: four a CU up to
    // heads of 128, then two and one); a batch of so many sequences that its
    // workgroups' search for their run would cost more than even runs gain has
    // one run each.
    const uint64_t resident = (attn->padded_dim <= 128u ? 4u : 512u / attn->padded_dim) *
                              (uint64_t)attn->ctx->num_cus;
    const uint64_t heads = (uint64_t)a.kv_heads * p.row_tiles;
    uint64_t chunks = std::min<uint64_t>(resident, kMaxPartials / 2u) / heads;
    // each sequence ends in a shorter run: on the average half a run more
    chunks = std::max(chunks - std::min<uint64_t>(chunks, a.num_seqs / 2u), chunks / 2u);
    p.chunks = a.num_seqs <= kMaxBalanced && chunks > 1u ? (uint32_t)chunks : 0u;
    const uint64_t pairs = a.kv_heads * ((uint64_t)p.chunks + a.num_seqs);
    const uint64_t blocks = p.row_tiles > 1u ? (pairs + 7u) / 8u * 8u * p.row_tiles : pairs;
    TSG_REQUIRE(blocks <= kMaxBlocks, TSG_ERR_UNSUPPORTED,
                "too many sequences and heads for one launch");
    p.pairs = (uint32_t)pairs;
    // the join's passes over a split's live rows, kJoinLoads splits a pass and way;
    // a tile of a run is done by one of the four waves
    const uint32_t pieces =
        std::min(a.seq_rows * a.group, kDecodeTileRows) * (attn->padded_dim / 8u);
    p.join_cost = (float)kWaves * (float)pieces / 256.0f / (float)kJoinLoads;
    p.part_o = attn->partials;
    p.part_ml = attn->partials + (uint64_t)kMaxPartials * 16u * attn->padded_dim;
    p.arrivals = attn->arrivals;
    const Variant v = variant_of(attn);
    hipLaunchKernelGGL(prefix ? v.shared : v.kernel, dim3((uint32_t)blocks), dim3(256), v.lds,
                       as_stream(stream), p);
    return check_launch("attn_decode");
}

}  // namespace tsg
