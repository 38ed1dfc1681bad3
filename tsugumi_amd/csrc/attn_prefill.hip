// attn_prefill.hip — attention of a prompt's rows, or of the next chunk of one,
// over the paged cache.
//
// A workgroup takes 128 rows of a sequence and key head, the heads of the group
// within the tokens (so a tile spans few positions and every key read serves
// the whole group), and goes through the keys they see, TK at a time: K and V
// tiles go from the pages into one of two LDS buffers while the other is
// computed on. Each of the four waves holds 32 rows: S^T = K Q^T and O^T =
// V^T P^T on 32 x 32 x 16 matrix instructions, Q, the weights and the sums in
// registers, V read from LDS transposed. Bound by the matrix instructions (2 D
// flop a pair each way) and, for narrow heads, by the exponentials beside them
// (16 cycles for 64 pairs against 0.25 D of matrix work).
//
// Measured on an MI355X: 8192 rows x 32 heads of 128 574-594 us over boxes, 926-958
// TFLOP/s (a large fp16 matrix product: 1306); the matrix units are busy 47 % of
// the time and the vector units 41 %, without bank conflicts.
//
// Where the rows are few and the keys many, the keys are split over several
// workgroups, and a second kernel joins their sums in the order of the splits.
//
// The keys that a group of decoded sequences shares are taken the same way, the group's rows in
// tiles of 128 (SHARED); the decode kernel joins these sums with each row's own keys'. 64
// sequences of 32 query and 8 key heads of 128 behind 16,000 keys, with 11 to 501 of their own: 36
// us, and 24 the decode kernel's.
#include "attn_internal.hpp"

namespace tsg {
namespace {

constexpr uint32_t kRows = kPrefillRows;  // of a workgroup
constexpr uint32_t kWaveRows = 32;        // of a wave
constexpr uint32_t kJoinRows = 8;         // rows a joining workgroup takes
constexpr float kFar = 1024.0f;           // a reference's logit in powers of two

struct PrefillArgs {
    AttnArgs a;
    float* part_o;   // [tile block][split][128][DP]
    float* part_ml;  // [tile block][split][128][2]
    uint32_t splits, min_tiles;
    uint32_t seq_tiles;  // row tiles of a sequence when its rows are uniform
    PrefixArgs x;        // for the keys that groups of sequences share
};

// Head elements a wave takes. At 512 a wave's sums and queries would fill all
// registers of a SIMD: two waves share the rows instead, each with one half of
// the elements, and add up their halves of the key products through LDS.
template <int DP>
constexpr uint32_t kWaveDim = DP <= 256 ? DP : DP / 2;
template <int DP>
constexpr uint32_t kThreads = 256u * (DP / kWaveDim<DP>);
template <int DP>
constexpr uint32_t prefill_lds_bytes() {
    return 2u * 2u * kTileKeys<DP> * DP * 2u + kRows * DP / 4u;  // + marks
}

// The row tile of workgroup `at` of a key head, counted from the last: sequences
// from the last to the first, a sequence's tiles from its last (most keys first).
// Uniform over the wave; kind 0 past the first. Starts that fall or pass the
// batch's rows make those before them meaningless: the workgroups after the tiles
// of the sequences behind the last such one leave NaN in all rows before those
// (kind 2; workgroup `tile` of `count`, rows under `seq`). Workgroup 0 looks at
// all starts and reports.
struct RowTile {
    uint32_t kind, seq, tile, count;
};
__device__ __forceinline__ RowTile find_tile(const PrefillArgs& p, uint32_t at, uint32_t blocks,
                                             bool check) {
    const AttnArgs& a = p.a;
    if (!a.row_starts)
        return RowTile{at / p.seq_tiles < a.num_seqs ? 1u : 0u, a.num_seqs - 1u - at / p.seq_tiles,
                       p.seq_tiles - 1u - at % p.seq_tiles, 0u};
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t behind = 0;  // tiles of the sequences behind these 64
    RowTile r{0u, 0u, 0u, 0u};
    for (uint32_t base = 0; base < a.num_seqs; base += 64u) {
        const bool live = base + lane < a.num_seqs;
        const uint32_t s = live ? a.num_seqs - 1u - (base + lane) : 0u;
        const uint32_t lo = live ? a.row_starts[s] : 0u, hi = live ? a.row_starts[s + 1u] : 0u;
        const uint64_t wrong = __ballot(lo > hi || hi > a.rows);
        if (check && wrong && lane == 0) report(a.error, kErrAttnRows);
        if (r.kind) continue;
        const int last_wrong = wrong ? __builtin_ctzll(wrong) : 64;
        const uint32_t tiles =
            (int)lane < last_wrong ? ((hi - lo) * a.group + kRows - 1u) / kRows : 0u;
        uint32_t sum = tiles;  // inclusive over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = (uint32_t)__shfl_up((int)sum, (unsigned)o, 64);
            if (lane >= (uint32_t)o) sum += v;
        }
        const uint64_t past = __ballot(behind + sum > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            const uint32_t end = behind + (uint32_t)__builtin_amdgcn_readlane((int)sum, l);
            r = RowTile{1u, a.num_seqs - 1u - (base + (uint32_t)l), end - 1u - at, 0u};
        } else {
            behind += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
            if (wrong)  // its end is where the next, right one starts
                r = RowTile{2u,
                            base == 0u && last_wrong == 0
                                ? a.rows
                                : (uint32_t)__builtin_amdgcn_readlane((int)hi, last_wrong),
                            at - behind, blocks - behind};
        }
        if (r.kind && !check) break;
    }
    return r;
}

// NaN in a key head's part of rows `first`, `first` + step, .. under `end`.
__device__ __forceinline__ void poison_rows(const AttnArgs& a, uint32_t kvh, uint32_t first,
                                            uint32_t step, uint32_t end) {
    const uint32_t pieces = a.group * a.dim / 8u;
    const uint32_t nan2 = 0x7E007E00u;
    for (uint64_t row = first; row < end; row += step)
        for (uint32_t n = threadIdx.x; n < pieces; n += blockDim.x)
            *reinterpret_cast<uint4*>(a.out + row * a.out_stride +
                                      (uint64_t)kvh * a.group * a.dim + 8u * n) =
                make_uint4(nan2, nan2, nan2, nan2);
}

// What a row tile's workgroups share: positions of its rows and the part of the
// key tiles that each split takes.
template <int DP>
struct TilePlan {
    uint32_t rows, r0, live;
    int32_t base, p_lo, p_hi;
    TileSpan span;
    uint32_t per, used;
};
template <int DP>
__device__ __forceinline__ TilePlan<DP> tile_plan(const PrefillArgs& p, const SeqRows& sr,
                                                  uint32_t tile) {
    const AttnArgs& a = p.a;
    TilePlan<DP> t;
    t.rows = sr.count * a.group;
    t.r0 = tile * kRows;
    t.live = t.rows - t.r0 < kRows ? t.rows - t.r0 : kRows;
    t.base = (int32_t)sr.length - (int32_t)sr.count;
    t.p_lo = t.base + (int32_t)(t.r0 / a.group);
    t.p_hi = t.base + (int32_t)((t.r0 + t.live - 1u) / a.group);
    t.span = tile_span<kTileKeys<DP>>(t.p_lo < 0 ? 0 : t.p_lo, t.p_hi, a.window, a.sinks);
    // the same run of key tiles for all of a sequence's rows: of its last rows'
    // span, so that a prompt's early rows, which see few keys, are not split
    const int32_t end = (int32_t)sr.length - 1;
    const int32_t end_lo = end - (int32_t)((t.rows < kRows ? t.rows : kRows) - 1u) / (int32_t)a.group;
    const uint32_t most =
        tile_span<kTileKeys<DP>>(end_lo < 0 ? 0 : end_lo, end, a.window, a.sinks).count;
    const uint32_t even = (most + p.splits - 1u) / p.splits;
    t.per = even > p.min_tiles ? even : p.min_tiles;
    // a window's span may begin one tile earlier in it than the last rows' does
    const uint32_t own = (t.span.count + p.splits - 1u) / p.splits;
    t.per = own > t.per ? own : t.per;
    const uint32_t used = (t.span.count + t.per - 1u) / t.per;
    t.used = used > 1u ? used : 1u;
    return t;
}

// Shared keys. A group's tokens that its sequences share: of the first one's pages, in whole
// key tiles; one sequence shares with none.
template <int DP>
__device__ __forceinline__ uint32_t shared_tokens(const AttnArgs& a, const PrefixArgs& x,
                                                  uint32_t g, uint32_t first_seq, uint32_t seqs) {
    if (seqs < 2u) return 0u;
    const uint32_t capacity = a.table_stride << a.page_shift, rows = seqs * a.seq_rows * a.group;
    const uint32_t length = a.lengths[first_seq];
    uint32_t n = x.shared[g];
    n = n < length ? n : length;
    n = n < capacity ? n : capacity;
    return share_pays(DP, seqs, rows, n) ? n / kShareTokens * kShareTokens : 0u;
}
// A group's row tiles, if it shares anything.
struct Group {
    uint32_t first_seq, seqs, tokens, tiles;
    bool wrong;  // its starts
};
template <int DP>
__device__ __forceinline__ Group group_of(const AttnArgs& a, const PrefixArgs& x, uint32_t g) {
    if (g >= x.num_groups) return Group{0u, 0u, 0u, 0u, false};
    const uint32_t lo = x.group_starts[g], hi = x.group_starts[g + 1u];
    if (lo > hi || hi > a.num_seqs) return Group{0u, 0u, 0u, 0u, true};
    const uint32_t tokens = lo < hi ? shared_tokens<DP>(a, x, g, lo, hi - lo) : 0u;
    const uint32_t tiles = tokens ? ((hi - lo) * a.seq_rows * a.group + kRows - 1u) / kRows : 0u;
    return Group{lo, hi - lo, tokens, tiles, false};
}
// All of a call's groups: the row tiles, and the splits that each one's keys may have, one
// workgroup a CU. Groups that share nothing, of no sequence or of one, count for nothing.
struct Groups {
    uint32_t tiles, splits;
    bool wrong;
};
template <int DP>
__device__ __forceinline__ Groups all_groups(const AttnArgs& a, const PrefixArgs& x) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t tiles = 0;
    bool wrong = false;
#pragma unroll 4
    for (uint32_t base = 0; base < x.num_groups; base += 64u) {
        const Group g = group_of<DP>(a, x, base + lane);
        wrong = wrong || g.wrong;
        tiles += g.tiles;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) tiles += (uint32_t)__shfl_xor((int)tiles, o, 64);
    tiles = __builtin_amdgcn_readfirstlane(tiles);
    uint32_t splits = tiles ? x.units / tiles : 1u;
    splits = splits < x.splits ? splits : x.splits;
    return Groups{tiles, splits ? splits : 1u, __ballot(wrong) != 0};
}
// Row tile `at` of all groups'.
struct GroupTile {
    uint32_t first_seq, seqs, tile, tokens;
};
template <int DP>
__device__ __forceinline__ GroupTile find_group_tile(const AttnArgs& a, const PrefixArgs& x,
                                                     uint32_t at) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t before = 0;
    for (uint32_t base = 0; base < x.num_groups; base += 64u) {
        const Group g = group_of<DP>(a, x, base + lane);
        uint32_t end = g.tiles;
#pragma unroll
        for (uint32_t o = 1; o < 64u; o <<= 1) {
            const uint32_t below = (uint32_t)__shfl_up((int)end, o, 64);
            end += lane >= o ? below : 0u;
        }
        const uint64_t behind = __ballot(before + end > at);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            const auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
            return GroupTile{of(g.first_seq), of(g.seqs), at - (before + of(end) - of(g.tiles)),
                             of(g.tokens)};
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
    }
    return GroupTile{0u, 0u, 0u, 0u};
}
// What the joining kernel needs to know of every sequence.
template <int DP>
__device__ __forceinline__ void write_info(const AttnArgs& a, const PrefixArgs& x) {
    const Groups all = all_groups<DP>(a, x);
    if (all.wrong && threadIdx.x == 0) report(a.error, kErrAttnGroups);
    for (uint32_t s = threadIdx.x; s < a.num_seqs; s += blockDim.x) {
        uint2 info = make_uint2(0u, all.splits * 2u + (all.wrong ? 1u : 0u));
        if (!all.wrong) {
            uint32_t lo = 0, hi = x.num_groups;  // the last group that starts at or before s
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2u;
                if (x.group_starts[mid] <= s) lo = mid + 1u;
                else hi = mid;
            }
            if (lo) {
                const uint32_t g = lo - 1u, first = x.group_starts[g], end = x.group_starts[g + 1u];
                if (s < end) info.x = shared_tokens<DP>(a, x, g, first, end - first);
            }
        }
        x.info[s] = info;
    }
}

// SHARED: the rows of a group of sequences over the keys that it shares, which leave
// partial sums.
template <int DP, bool E4M3, bool FULL, bool SHARED = false>
__global__ __launch_bounds__(kThreads<DP>, 2) void prefill_kernel(PrefillArgs p) {
    constexpr uint32_t TK = kTileKeys<DP>;
    constexpr uint32_t DW = kWaveDim<DP>, THREADS = kThreads<DP>, SHARE = DP / DW;
    constexpr uint32_t NS = DW / 16, NB = DW / 32;  // key-product steps, value blocks of a wave
    constexpr uint32_t ROW = DP * 2u;               // bytes of a key's row in LDS
    constexpr uint32_t CPR = DP / 8u;               // 16-byte chunks of it
    constexpr uint32_t TILE = TK * ROW;
    constexpr uint32_t KW = TK / (4u * SHARE);      // keys a wave stages
    constexpr bool DMA = !E4M3 && FULL;
    extern __shared__ __align__(16) uint8_t smem[];
    const AttnArgs& a = p.a;

    // of shared keys: the tiles of a split beside each other, workgroups without one behind all
    uint32_t split = SHARED ? 0u : blockIdx.y, at = blockIdx.x / a.kv_heads;
    const uint32_t kvh = blockIdx.x % a.kv_heads;
    uint32_t s = 0;
    SeqRows sr{};
    TilePlan<DP> t{};
    uint32_t tile_first = 0, tile_end = 0, shared = 0;
    if constexpr (SHARED) {
        if (blockIdx.x == gridDim.x - 1u) {
            write_info<DP>(a, p.x);
            return;
        }
        const Groups all = all_groups<DP>(a, p.x);
        if (all.wrong || at >= all.tiles * all.splits) return;
        split = at / all.tiles;
        const GroupTile gt = find_group_tile<DP>(a, p.x, at % all.tiles);
        s = gt.first_seq;  // its page table
        shared = gt.tokens;
        const PrefixSplit ps = prefix_split(p.x, all.splits, shared / TK);
        if (split >= ps.used) return;
        t.rows = gt.seqs * a.seq_rows * a.group;
        t.r0 = gt.tile * kRows;
        t.live = t.rows - t.r0 < kRows ? t.rows - t.r0 : kRows;
        t.used = 2u;  // partial sums
        tile_first = split * ps.per;
        tile_end = tile_first + ps.per;
    } else {
        const RowTile rt = find_tile(p, at, gridDim.x / a.kv_heads, at == 0u && split == 0u);
        if (rt.kind != 1u) {
            if (rt.kind == 2u && split == 0u) poison_rows(a, kvh, rt.tile, rt.count, rt.seq);
            return;
        }
        s = rt.seq;
        const uint32_t capacity = a.table_stride << a.page_shift;
        sr = seq_rows(a.row_starts, a.lengths, s, a.seq_rows, a.rows, capacity);
        t = tile_plan<DP>(p, sr, rt.tile);
        if (split >= t.used) return;
        tile_first = split * t.per;
        tile_end = tile_first + t.per < t.span.count ? tile_first + t.per : t.span.count;
        if (sr.bad) tile_end = tile_first;
    }
    // position of row r of the workgroup's: of its own keys the last, of shared ones at most
    const auto row_pos = [&](uint32_t r) -> int32_t {
        if constexpr (SHARED) {
            const uint32_t token = (t.r0 + r) / a.group, seq = s + token / a.seq_rows;
            const uint32_t capacity = a.table_stride << a.page_shift, length = a.lengths[seq];
            const int32_t pos = (int32_t)(length < capacity ? length : capacity) -
                                (int32_t)a.seq_rows + (int32_t)(token % a.seq_rows);
            return pos < (int32_t)shared ? pos : (int32_t)shared - 1;
        } else {
            return t.base + (int32_t)((t.r0 + r) / a.group);
        }
    };

    const uint32_t lane = threadIdx.x & 63u, i32 = lane & 31u, h = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // the wave's rows; lane i32 of both halves holds row i32 of them
    const uint32_t w0 = (wave & 3u) * kWaveRows;  // within the tile
    const uint32_t d0 = (wave >> 2) * DW;         // its first head element
    const bool wave_live = w0 < t.live;
    const uint32_t w_last = w0 + 31u < t.live ? w0 + 31u : t.live - 1u;
    const uint32_t row = t.r0 + (w0 + i32 < t.live ? w0 + i32 : t.live - 1u);
    const uint32_t tok = row / a.group;
    const int32_t pos = row_pos(row - t.r0);
    int32_t p_lo, p_hi;
    if constexpr (SHARED) {  // of the workgroup's rows, of sequences of any lengths
        const uint32_t r1 = lane < t.live ? lane : t.live - 1u;
        const uint32_t r2 = lane + 64u < t.live ? lane + 64u : t.live - 1u;
        const int32_t p1 = row_pos(r1), p2 = row_pos(r2);
        p_lo = p1 < p2 ? p1 : p2;
        p_hi = p1 < p2 ? p2 : p1;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const int32_t lo = __shfl_xor(p_lo, o, 64), hi = __shfl_xor(p_hi, o, 64);
            p_lo = p_lo < lo ? p_lo : lo;
            p_hi = p_hi > hi ? p_hi : hi;
        }
        p_lo = __builtin_amdgcn_readfirstlane(p_lo);
        p_hi = __builtin_amdgcn_readfirstlane(p_hi);
        t.p_lo = p_lo;
        t.p_hi = p_hi;
        t.span = tile_span<TK>(0, p_hi, 0u, 0u);
        tile_end = tile_end < t.span.count ? tile_end : t.span.count;
        sr.first = s * a.seq_rows;
    } else {
        p_lo = t.base + (int32_t)((t.r0 + (wave_live ? w0 : 0u)) / a.group);
        p_hi = t.base + (int32_t)((t.r0 + w_last) / a.group);
    }
    const uint32_t q_head = kvh * a.group + row % a.group;
    const uint16_t* q = a.q + (uint64_t)(sr.first + tok) * a.q_stride + (uint64_t)q_head * a.dim;
    h8_t qf[NS];  // step st takes, from lane half h, elements 16 st + 8 h ..
#pragma unroll
    for (uint32_t st = 0; st < NS; ++st) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (FULL || d0 + 16u * st + 8u * h < a.dim)
            u = load_query(q + d0 + 16u * st + 8u * h, a.q_sign);
        qf[st] = __builtin_bit_cast(h8_t, u);
    }

    // ------------------------------------------------------------- staging
    // Key t's row: chunk c of K lies at c ^ key_swizzle(t), of V at c ^
    // value_swizzle(t): 16 keys' equal chunks, and the 8 keys of a transposing
    // read, lie in different banks.
    const auto key_swizzle = [](uint32_t k) { return DP >= 128 ? k & 15u : (k >> 1) & 7u; };
    const auto value_swizzle = [](uint32_t k) {
        return 2u * (DP >= 128 ? ((k & 3u) << 1) | ((k >> 2) & 1u)
                               : (((k >> 1) & 1u) << 1) | ((k >> 2) & 1u));
    };
    const uint32_t* table = a.table + (uint64_t)s * a.table_stride;
    const uint32_t page_mask = (1u << a.page_shift) - 1u;
    const uint32_t last_page = t.p_hi < 0 ? 0u : (uint32_t)t.p_hi >> a.page_shift;
    const uint64_t head_off = (uint64_t)kvh * a.head_stride;
    bool bad = false;
    // byte offset in the pools of the first key that this wave stages
    const auto wave_offset = [&](uint32_t idx) -> uint64_t {
        const uint32_t k0 = t.span.key_tile(idx) * TK + wave * KW;
        const uint32_t want = k0 >> a.page_shift;
        uint32_t page = scalar_load(table + (want < last_page ? want : last_page));
        if (page >= a.num_pages) {
            bad = bad || keys_seen<KW>(k0, t.p_lo, t.p_hi, a.window, a.sinks);
            page = 0u;
        }
        return page * a.page_stride + head_off + (uint64_t)(k0 & page_mask) * a.token_stride;
    };
    constexpr uint32_t SRC = E4M3 ? CPR / 2u : CPR;  // 16-byte chunks of a cache row
    constexpr uint32_t KPI = 64u / SRC;              // keys of one load instruction
    constexpr uint32_t NL = KW / KPI;                // loads of K (and of V) a tile
    static_assert(NL >= 1u && KW % KPI == 0u, "a wave's keys are whole load instructions");
    const uint32_t l_key = lane / SRC, l_chunk = lane % SRC, l_row = l_key * a.token_stride;
    const auto k_tile = [&](uint32_t buf) { return smem + buf * 2u * TILE; };
    const auto v_tile = [&](uint32_t buf) { return smem + buf * 2u * TILE + TILE; };
    uint4 kst[DMA ? 1 : NL], vst[DMA ? 1 : NL];
    // The wave's keys of a tile, from byte `off` of a pool: to LDS at once, or to
    // registers (begin) and from there, as fp16, to LDS (end).
    const auto stage_begin = [&](const uint8_t* pool, uint64_t off, uint8_t* to, auto swizzle,
                                 uint4* regs) {
        if constexpr (DMA) {
            const uint32_t lds = (uint32_t)(uintptr_t)to + wave * KW * ROW;
            // offsets are formed here each time (opaque lane): hoisted they would be
            // spilled, and a reload's wait would drain the loads under way
            uint32_t c = l_chunk;
            asm("" : "+v"(c));
#pragma unroll
            for (uint32_t n = 0; n < NL; ++n)
                dma16(pool + (off + n * KPI * a.token_stride),
                      l_row + 16u * (c ^ swizzle(wave * KW + n * KPI + l_key)), lds + n * KPI * ROW);
        } else {
            const bool in = FULL || l_chunk * 16u < a.dim * (E4M3 ? 1u : 2u);
#pragma unroll
            for (uint32_t n = 0; n < NL; ++n) {
                const uint4 x = *reinterpret_cast<const uint4*>(
                    pool + (off + n * KPI * a.token_stride) + (l_row + (in ? 16u * l_chunk : 0u)));
                regs[n] = in ? x : make_uint4(0, 0, 0, 0);
            }
        }
    };
    const auto stage_end = [&](uint8_t* to, auto swizzle, const uint4* regs) {
        if constexpr (!DMA) {
#pragma unroll
            for (uint32_t n = 0; n < NL; ++n) {
                const uint32_t k = wave * KW + n * KPI + l_key, z = swizzle(k);
                if constexpr (E4M3) {
                    const uint2 x0 = e4m3x4_to_f16(regs[n].x), x1 = e4m3x4_to_f16(regs[n].y);
                    const uint2 x2 = e4m3x4_to_f16(regs[n].z), x3 = e4m3x4_to_f16(regs[n].w);
                    *reinterpret_cast<uint4*>(to + k * ROW + 16u * ((2u * l_chunk) ^ z)) =
                        make_uint4(x0.x, x0.y, x1.x, x1.y);
                    *reinterpret_cast<uint4*>(to + k * ROW + 16u * ((2u * l_chunk + 1u) ^ z)) =
                        make_uint4(x2.x, x2.y, x3.x, x3.y);
                } else {
                    *reinterpret_cast<uint4*>(to + k * ROW + 16u * (l_chunk ^ z)) = regs[n];
                }
            }
        }
    };
    const auto k_begin = [&](uint64_t off, uint32_t buf) {
        stage_begin(a.k, off, k_tile(buf), key_swizzle, kst);
    };
    const auto v_begin = [&](uint64_t off, uint32_t buf) {
        stage_begin(a.v, off, v_tile(buf), value_swizzle, vst);
    };
    const auto k_end = [&](uint32_t buf) { stage_end(k_tile(buf), key_swizzle, kst); };
    const auto v_end = [&](uint32_t buf) { stage_end(v_tile(buf), value_swizzle, vst); };
    // every wave's part of the tiles is in LDS, and every wave done with the last
    const auto staged = [&] {
        wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // ------------------------------------------------------------- compute
    f16v_t o[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][e] = 0.0f;
    float m = kNoKey, l = 0.0f;
    // (x - m) scale_log2 + bias as one multiply-add, with m's part rounded by
    // itself (by 2^-14 at most), or, far from zero, of the difference
    float shift = __builtin_fmaf(-kNoKey, a.scale_log2, kWeightBias);
    bool far = false;  // some row of the wave's is
    // Accumulator register e of lane half h is key 8 (e / 4) + 4 h + e % 4 of 32;
    // registers 8 ss .. 8 ss + 7 are the lane's eight of the second operand of
    // V^T P^T's step ss, whose first operand comes in two transposing reads.
    const uint32_t i16 = lane & 15u, tr_key = 4u * h + (i16 >> 2);
    const uint32_t k_at = i32 * ROW + 2u * d0, k_swz = key_swizzle(i32);
    const uint32_t v_at = tr_key * ROW + 2u * d0 + 8u * (i16 & 3u);
    const uint32_t v_chunk = (2u * ((lane >> 4) & 1u)) ^ value_swizzle(tr_key);

    // the wave's rows against a tile's keys, in steps
    constexpr uint32_t N = TK / 32u;
    const auto products = [&](uint8_t* kb, f16v_t (&x)[N]) {
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[u][e] = 0.0f;
#pragma unroll
        for (uint32_t st = 0; st < NS; ++st)
#pragma unroll
            for (uint32_t u = 0; u < N; ++u) {
                const h8_t kf = *reinterpret_cast<const h8_t*>(
                    kb + u * 32u * ROW + k_at + 16u * ((2u * st + h) ^ k_swz));
                x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[st], x[u], 0, 0, 0);
            }
        if constexpr (SHARE == 2u) {  // through the K tile, once every wave is done with it
            static_assert(N == 1u && 2u * 4u * 64u * 64u <= TILE, "the sums fit the K tile");
            lds_barrier();
            f4_t* mine = reinterpret_cast<f4_t*>(kb) + wave * 256u + lane;
            const f4_t* other = reinterpret_cast<const f4_t*>(kb) + (wave ^ 4u) * 256u + lane;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                mine[64 * k] = f4_t{x[0][4 * k], x[0][4 * k + 1], x[0][4 * k + 2], x[0][4 * k + 3]};
            lds_barrier();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f4_t y = other[64 * k];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[0][4 * k + e] += y[e];
            }
        }
    };
    const auto mask = [&](f16v_t (&x)[N], uint32_t key0) {
        if (tile_seen_whole<TK>(key0, p_lo, p_hi, a.window, a.sinks)) return;
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!key_seen((int32_t)(key0 + 32u * u + 8u * (e / 4) + 4u * h + e % 4), pos,
                              a.window, a.sinks))
                    x[u][e] = -__builtin_inff();
    };
    const auto move_reference = [&](const f16v_t (&x)[N]) {
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, x[u][e]);
        if (__ballot((top - m) * a.scale_log2 > kMaxLag)) {
            const float mn = fmaxf(m, max_across32(top));
            const float alpha = __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
            m = mn;
            const bool row_far = fabsf(m * a.scale_log2) >= kFar && m != kNoKey;
            shift = row_far ? kWeightBias : __builtin_fmaf(-m, a.scale_log2, kWeightBias);
            far = __ballot(row_far) != 0;
            l *= alpha;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) o[b] *= alpha;
        }
    };
    const auto weights = [&](f16v_t (&x)[N], h8_t (&w)[N][2]) {
        if (far) {
            const float sub = shift == kWeightBias ? m : 0.0f;
#pragma unroll
            for (uint32_t u = 0; u < N; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[u][e] -= sub;
        }
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const h2_t two = weight_pair(__builtin_fmaf(x[u][e], a.scale_log2, shift),
                                             __builtin_fmaf(x[u][e + 1], a.scale_log2, shift));
                l = dot2(two, h2_t{1, 1}, l);
                w[u][e / 8][e % 8] = two[0];
                w[u][e / 8][e % 8 + 1] = two[1];
            }
    };
    const auto add_values = [&](const h8_t (&w)[N][2], const uint8_t* vb) {
#pragma unroll
        for (uint32_t u = 0; u < N; ++u)
#pragma unroll
            for (uint32_t ss = 0; ss < 2u; ++ss)
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    const uint8_t* at_v =
                        vb + (u * 32u + 16u * ss) * ROW + v_at + 16u * ((4u * b) ^ v_chunk);
                    const uint2 lo = lds_read_tr(at_v), hi = lds_read_tr(at_v + 8u * ROW);
                    const h8_t vf = __builtin_bit_cast(h8_t, make_uint4(lo.x, lo.y, hi.x, hi.y));
                    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, w[u][ss], o[b], 0, 0, 0);
                }
    };

    // A tile that some row sees a part of: an infinity or NaN in its V would
    // make NaN of the weight 0 of a row that does not see its key. They are
    // taken out of LDS and noted in `marks` (two bits, +inf and -inf, NaN both,
    // for each element of the rows that see the key), which go onto the sums at
    // the end.
    uint32_t* marks = reinterpret_cast<uint32_t*>(smem + 4u * TILE);  // [row][DP / 16]
    bool marked = false;
    const auto take_out = [&](uint8_t* vb, uint32_t key0) {
        bool found = false;
#pragma unroll 1
        for (uint32_t c = threadIdx.x; c < TK * CPR; c += THREADS) {
            uint4* at = reinterpret_cast<uint4*>(vb + 16u * c);
            if (!keys_seen<1>(key0 + c / CPR, t.p_lo, t.p_hi, a.window, a.sinks)) {
                *at = make_uint4(0, 0, 0, 0);  // no row's: it may hold anything
                continue;
            }
            const uint4 v = *at;
            found = found || (not_finite<false>(v.x) | not_finite<false>(v.y) |
                              not_finite<false>(v.z) | not_finite<false>(v.w)) != 0u;
        }
        if (!__syncthreads_or(found)) return;
        if (!marked) {
            for (uint32_t n = threadIdx.x; n < kRows * DP / 16u; n += THREADS) marks[n] = 0u;
            marked = true;
            __syncthreads();
        }
#pragma unroll 1
        for (uint32_t n = threadIdx.x; n < TK * DP; n += THREADS) {
            uint16_t* v = reinterpret_cast<uint16_t*>(vb) + n;
            const uint32_t bits = *v;
            if ((bits & 0x7C00u) != 0x7C00u) continue;
            *v = 0;
            const uint32_t k = n / DP, e = n % DP;
            const uint32_t dim = 8u * ((e / 8u) ^ value_swizzle(k)) + e % 8u;
            const uint32_t mark = (bits & 0x3FFu ? 3u : bits & 0x8000u ? 2u : 1u) << (2u * (dim & 15u));
#pragma unroll 1
            for (uint32_t r = 0; r < t.live; ++r)
                if (key_seen((int32_t)(key0 + k), row_pos(r), a.window, a.sinks))
                    atomicOr(marks + r * (DP / 16u) + dim / 16u, mark);
        }
        __syncthreads();
    };

    const auto key0_of = [&](uint32_t idx) { return t.span.key_tile(idx) * TK; };
    // a tile that not all rows of the workgroup see whole
    const auto clean_values = [&](uint32_t idx, uint8_t* vb) {
        if (!tile_seen_whole<TK>(key0_of(idx), t.p_lo, t.p_hi, a.window, a.sinks))
            take_out(vb, key0_of(idx));
    };
    if (tile_first < tile_end) {
        const uint64_t off = wave_offset(tile_first);
        k_begin(off, 0u);
        v_begin(off, 0u);
        k_end(0u);
        v_end(0u);
    }
    for (uint32_t idx = tile_first; idx < tile_end; ++idx) {
        const uint32_t buf = (idx - tile_first) & 1u;
        const bool more = idx + 1u < tile_end;
        staged();
        if (more) {
            const uint64_t off = wave_offset(idx + 1u);
            k_begin(off, buf ^ 1u);
            v_begin(off, buf ^ 1u);
        }
        clean_values(idx, v_tile(buf));
        const uint32_t key0 = key0_of(idx);
        // waves that share rows meet inside; every wave goes in
        if (SHARE == 2u || (wave_live && keys_seen<TK>(key0, p_lo, p_hi, a.window, a.sinks))) {
            f16v_t x[N];
            h8_t w[N][2];
            products(k_tile(buf), x);
            mask(x, key0);
            move_reference(x);
            weights(x, w);
            add_values(w, v_tile(buf));
        }
        if (more) {
            k_end(buf ^ 1u);
            v_end(buf ^ 1u);
        }
    }

    // a page past the pool: the tile's rows are NaN, whichever wave met it
    uint32_t* flag = reinterpret_cast<uint32_t*>(smem);
    __syncthreads();
    if (threadIdx.x == 0) *flag = 0u;
    __syncthreads();
    if (lane == 0 && (bad || sr.bad)) {
        report(a.error, sr.bad ? sr.bad : kErrAttnPage);
        *flag = 1u;
    }
    __syncthreads();
    l = sum_across32(l);
    if (*flag) l = __builtin_nanf("");
    if (w0 + i32 >= t.live) return;
    if (marked) {
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t dim = d0 + 32u * b + 8u * (e / 4) + 4u * h + e % 4;
                const uint32_t mark =
                    marks[(w0 + i32) * (DP / 16u) + dim / 16u] >> (2u * (dim & 15u));
                if (mark & 1u) o[b][e] += __builtin_inff();
                if (mark & 2u) o[b][e] -= __builtin_inff();
            }
    }

    // lane half h holds elements 32 b + 8 k + 4 h .. + 3 of its row
    if (!SHARED && t.used == 1u) {
        const float inv = row_inverse(l, pos, a.v_scale);
        uint16_t* out = a.out + (uint64_t)(sr.first + tok) * a.out_stride + (uint64_t)q_head * a.dim;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                const uint32_t e = d0 + 32u * b + 8u * k + 4u * h;
                if (!FULL && e >= a.dim) continue;
                uint2 u;
                u.x = (uint32_t)f32_to_f16(o[b][4 * k] * inv) |
                      ((uint32_t)f32_to_f16(o[b][4 * k + 1] * inv) << 16);
                u.y = (uint32_t)f32_to_f16(o[b][4 * k + 2] * inv) |
                      ((uint32_t)f32_to_f16(o[b][4 * k + 3] * inv) << 16);
                *reinterpret_cast<uint2*>(out + e) = u;
            }
    } else {
        const uint64_t slot =
            SHARED ? (uint64_t)(kvh * p.x.splits + split) * p.x.rows +
                         s * a.seq_rows * a.group + t.r0 + w0 + i32
                   : ((uint64_t)blockIdx.x * p.splits + split) * kRows + w0 + i32;
        float* part_ml = SHARED ? p.x.part_ml : p.part_ml;
        float* dst = (SHARED ? p.x.part_o : p.part_o) + slot * DP;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                *reinterpret_cast<float4*>(dst + d0 + 32u * b + 8u * k + 4u * h) = make_float4(
                    o[b][4 * k], o[b][4 * k + 1], o[b][4 * k + 2], o[b][4 * k + 3]);
        if (h == 0 && d0 == 0) *reinterpret_cast<float2*>(part_ml + slot * 2u) = make_float2(m, l);
    }
}

// Adds up the splits' sums of a row tile, kJoinRows rows a workgroup: `ways`
// neighbouring lanes share an 8-element piece, each takes every ways-th split,
// in order, from loads that go out together.
template <int DP>
__global__ __launch_bounds__(256) void prefill_join_kernel(PrefillArgs p) {
    constexpr uint32_t C8 = DP / 8u, PIECES = kJoinRows * C8;
    const AttnArgs& a = p.a;
    const uint32_t kvh = blockIdx.x % a.kv_heads;
    const RowTile rt = find_tile(p, blockIdx.x / a.kv_heads, gridDim.x / a.kv_heads, false);
    if (rt.kind != 1u) return;
    const SeqRows sr = seq_rows(a.row_starts, a.lengths, rt.seq, a.seq_rows, a.rows,
                                a.table_stride << a.page_shift);
    const TilePlan<DP> t = tile_plan<DP>(p, sr, rt.tile);
    if (t.used == 1u || blockIdx.y * kJoinRows >= t.live) return;
    uint32_t ways = 1u;
    while (ways < t.used && 2u * ways * PIECES <= 256u) ways *= 2u;
    const uint32_t way = threadIdx.x & (ways - 1u);
    for (uint32_t n = 0; n < PIECES; n += 256u / ways) {
        const uint32_t piece = n + threadIdx.x / ways;
        const uint32_t r = blockIdx.y * kJoinRows + piece / C8, c = piece % C8;
        const bool in = piece < PIECES && r < t.live && 8u * c < a.dim;
        const uint64_t slot = (uint64_t)blockIdx.x * p.splits * kRows + (in ? r : 0u);
        float m = kNoKey, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f;
#pragma unroll 4
        for (uint32_t w = way; w < t.used; w += ways) {
            const uint64_t at = slot + (uint64_t)w * kRows;
            const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2u);
            const f4_t* src = reinterpret_cast<const f4_t*>(p.part_o + at * DP + 8u * c);
            const f4_t lo = src[0], hi = src[1];
            const float mn = fmaxf(m, ml.x);
            const float f0 = __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
            const float f1 = __builtin_amdgcn_exp2f((ml.x - mn) * a.scale_log2);
            m = mn;
            sum = sum * f0 + ml.y * f1;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f0 + (e < 4 ? lo[e & 3] : hi[e & 3]) * f1;
        }
        for (uint32_t o = 1; o < ways; o <<= 1) {
            const float m2 = __shfl_xor(m, (int)o, 64), mn = fmaxf(m, m2);
            const float f0 = __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
            const float f1 = __builtin_amdgcn_exp2f((m2 - mn) * a.scale_log2);
            m = mn;
            sum = sum * f0 + __shfl_xor(sum, (int)o, 64) * f1;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f0 + __shfl_xor(acc[e], (int)o, 64) * f1;
        }
        if (!in || way != 0u) continue;
        const uint32_t tok = (t.r0 + r) / a.group;
        const float inv = row_inverse(sum, t.base + (int32_t)tok, a.v_scale);
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = (uint32_t)f32_to_f16(acc[2 * e] * inv) |
                   ((uint32_t)f32_to_f16(acc[2 * e + 1] * inv) << 16);
        *reinterpret_cast<uint4*>(a.out + (uint64_t)(sr.first + tok) * a.out_stride +
                                  (uint64_t)(kvh * a.group + (t.r0 + r) % a.group) * a.dim +
                                  8u * c) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

typedef void (*PrefillKernel)(PrefillArgs);

template <int DP, bool SHARED>
PrefillKernel kernel_of(bool e4m3, bool full) {
    if (e4m3)
        return full ? prefill_kernel<DP, true, true, SHARED> : prefill_kernel<DP, true, false, SHARED>;
    return full ? prefill_kernel<DP, false, true, SHARED> : prefill_kernel<DP, false, false, SHARED>;
}

struct Variant {
    PrefillKernel kernel, join, shared;
    uint32_t threads, lds, tile_keys;
};
template <int DP>
Variant variant(bool e4m3, bool full) {
    return {kernel_of<DP, false>(e4m3, full), prefill_join_kernel<DP>, kernel_of<DP, true>(e4m3, full),
            kThreads<DP>, prefill_lds_bytes<DP>(), kTileKeys<DP>};
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

tsg_status prepare_prefill(const tsg_attn* attn) {
    const Variant v = variant_of(attn);
    for (PrefillKernel kernel : {v.kernel, v.shared})
        TSG_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)v.lds));
    return TSG_OK;
}

tsg_status launch_prefixes(const tsg_attn* attn, const AttnArgs& a, PrefixArgs* x,
                           tsg_stream stream) {
    const Variant v = variant_of(attn);
    const uint64_t rows = (uint64_t)a.rows * a.group;
    TSG_REQUIRE(rows * a.kv_heads <= kMaxPrefixRows, TSG_ERR_DECLINED,
                "too many rows and query heads for the plan's scratch: tsg_attn_decode");
    // One workgroup a CU, of at least four key tiles: with two, the partial sums' way through
    // memory costs what the shorter runs gain (both launches, 250 keys a sequence of its own
    // behind 16,000: 64 sequences 58 us with one and with two, with heads of 256 72 and 86, 32
    // sequences 54 and 64, 8 32 and 35; 8 groups of 8 behind 4096, 200 of their own, 49 and 48).
    // How many tiles there are, the device sees: a group that shares has two sequences at least,
    // and may end inside a tile.
    const uint64_t most = rows / kRows + std::min(x->num_groups, a.num_seqs / 2u);
    const uint64_t capacity_tiles =
        (((uint64_t)a.table_stride << a.page_shift) + v.tile_keys - 1u) / v.tile_keys;
    x->min_tiles = 4u;
    x->units = std::max<uint32_t>(attn->ctx->num_cus * 256u / v.threads / a.kv_heads, 1u);
    uint64_t splits = (capacity_tiles + x->min_tiles - 1u) / x->min_tiles;
    splits = std::min<uint64_t>(splits, kMaxPrefixRows / (rows * a.kv_heads));
    x->splits = (uint32_t)std::max<uint64_t>(splits, 1u);
    x->rows = (uint32_t)rows;
    const uint64_t row0 = kMaxPartials * (uint64_t)kDecodeTileRows, dp = attn->padded_dim;
    x->part_o = attn->partials + row0 * (dp + 2u);
    x->part_ml = x->part_o + kMaxPrefixRows * dp;
    x->info = reinterpret_cast<uint2*>(x->part_ml + kMaxPrefixRows * 2u);
    PrefillArgs p{};
    p.a = a;
    p.x = *x;
    const uint64_t units = std::max<uint64_t>(x->units, most);  // few: the rows bound them
    hipLaunchKernelGGL(v.shared, dim3((uint32_t)(a.kv_heads * units) + 1u), dim3(v.threads), v.lds,
                       as_stream(stream), p);
    return check_launch("attn_prefixes");
}

tsg_status launch_prefill(const tsg_attn* attn, const AttnArgs& a, tsg_stream stream) {
    const Variant v = variant_of(attn);
    PrefillArgs p{};
    p.a = a;
    p.seq_tiles = a.row_starts ? 0u : (uint32_t)(((uint64_t)a.seq_rows * a.group + kRows - 1u) / kRows);
    // row starts: every sequence may end inside a tile
    const uint64_t tiles = a.row_starts
                               ? (uint64_t)a.rows * a.group / kRows + std::min(a.num_seqs, a.rows)
                               : (uint64_t)a.num_seqs * p.seq_tiles;
    const uint64_t blocks = tiles * a.kv_heads;
    TSG_REQUIRE(blocks * (v.threads / 256u) <= kMaxBlocks, TSG_ERR_UNSUPPORTED,
                "too many rows and heads for one launch");
    // Splits where the row tiles are fewer than the workgroups the card holds:
    // up to twice as many, since a prompt's tiles are uneven (2011 rows of 512-wide
    // heads in 252 workgroups 167 us, in up to 504 147), of at least four key
    // tiles (67 rows over 967 keys 24.0 us, of at least two 25.1).
    const uint64_t capacity_tiles =
        (((uint64_t)a.table_stride << a.page_shift) + v.tile_keys - 1u) / v.tile_keys;
    p.min_tiles = 4u;
    const uint64_t resident = 2u * (uint64_t)attn->ctx->num_cus * 256u / v.threads;
    uint64_t splits = 2u * resident / blocks;
    splits = std::min(splits, (capacity_tiles + p.min_tiles - 1u) / p.min_tiles);
    splits = std::min<uint64_t>(splits, kMaxPrefillPartials / blocks);
    p.splits = (uint32_t)std::max<uint64_t>(splits, 1u);
    p.part_o = attn->partials;
    p.part_ml = attn->partials + (uint64_t)kMaxPrefillPartials * kRows * attn->padded_dim;
    hipLaunchKernelGGL(v.kernel, dim3((uint32_t)blocks, p.splits), dim3(v.threads), v.lds,
                       as_stream(stream), p);
    if (tsg_status s = check_launch("attn_prefill")) return s;
    if (p.splits > 1u) {
        hipLaunchKernelGGL(v.join, dim3((uint32_t)blocks, kRows / kJoinRows), dim3(256), 0,
                           as_stream(stream), p);
        return check_launch("attn_prefill_join");
    }
    return TSG_OK;
}

}  // namespace tsg
