// Latent attention, absorbed form over a paged cache (gfx950): all heads of a sequence read the same 576-wide token rows, whose
// first 512 values are keys and values at once.
//
// The query rows (token, head) of a sequence are taken in groups of up to 64 (two row tiles of 32) and the keys in tiles of 32.
// The work is cut along the keys: a launch of about one workgroup a CU, each with an equal run of key tiles through the packed
// sequences (all groups of a sequence side by side, so that their reads of the same keys meet in one L2), and with a shared
// prefix some of the workgroups walk its tiles for groups of all rows of the batch.  Every workgroup finds its run from the
// lengths on the device.  A run that holds a sequence whole writes its output; parts are left in the workspace in fp32 and
// joined by a second kernel:  o = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s.
//
// 8 waves, two a SIMD, of two kinds.  In the step of tile j the score waves 0 .. 3 (row tile w % 2, keys 16 (w / 2) .. + 15; their
// queries in 144 registers) compute its scores and leave its weights in LDS, while the value waves 4 .. 7 add tile j - 1 to values
// 128 (w - 4) .. + 127 of all rows (128 accumulators) and bring tile j + 2 straight into LDS (36 KiB a tile, four tiles): matrix
// instructions of one kind run beside the softmax, the waits and the address arithmetic of the other.  One barrier a tile.
// Scores come from 16x16x32 instructions (keys as rows), so that every key fragment read serves two of them; values from
// 32x32x16 with one fragment for both row tiles.
// With one row tile a group (RT = 1) a score wave has rows 16 (w % 2) .. + 15 of it and everything of a row is there once.
//
// Bound: with many rows of few sequences the step itself.  The two products are 576 and 512 cycles of a SIMD's matrix core a tile, a step
// takes about 2200 (busy cycles of a CU over the units it walks): scores, maxima across lanes, weights through LDS and a barrier
// follow one another, so the matrix cores are busy 48 % and LDS 33 % of the time.  Calls with their join, one after the other on inputs that
// change: 16 sequences of 6000 to 9900 tokens, 8 draft tokens, 96 heads (drafts, fp16) 221 to 232 us, 0.91 to 0.96 PFLOP/s; 64 sequences of
// 32 heads behind 32768 shared tokens 156 us, 0.95 PFLOP/s, of 64 heads 324.  With a row tile or two a sequence HBM: 64 ragged sequences of
// 64 heads 126 to 128 us, 4.3 TB/s, of 32 heads 109 to 115.  One sequence of 4097 tokens, 12 heads: 13.9 us from a graph,
// 9.0 of it this kernel (lengths and cut 2.2, queries and first tile 2.0, three tiles and the end 3) and 4.5 the join.
// A cache in 4 bits (Q4) stays in 4 bits in LDS (13 KiB a tile, eight tiles, brought seven ahead); both kinds of waves widen what they
// multiply, in registers: a score wave its 16 keys between its products, a value wave the next tile's values while it multiplies this
// one's.  Bound by the step: a wave has some 80 instructions for that in it beside its products, and the SIMD's two (three) waves' vector
// instructions (46 %) and products (43 %) rarely run side by side.  So many rows take as long as over 16 bits or a little longer: drafts 225
// to 231 us, 32 heads behind the prefix 158 to 161, 64 heads 336 to 342; few rows less: 64 ragged sequences of 64 heads 84 to 92, of 32 heads
// 62 to 72 (3.0 TB/s; this kernel alone, on a cache that stays in L3, 53 us and 3.6 TB/s).  Pages that are no multiple of 8 tokens (not EVEN:
// an address a token): drafts 241, 64 heads behind the prefix 371, 32 heads ragged 73.
// What a segment keeps from before the loops is spilled, and its reload waits for every load under way: addresses are found where they are
// needed (drafts 246 us with the join before, 226 so).  Nothing is spilled in a vector register but by the form for two row tiles that is not
// EVEN: 1 in bf16, 4 in fp16.
// Forms before it (64 ragged sequences of 32 heads / drafts / 64 heads behind the prefix, without the join): 16-bit tiles made in LDS by waves of their own 78 / 284 / 447 us, made by the value waves 69 / 261 / 396.  Two tiles a
// step with one row tile: 62 against 64, and 12.0 against 10.3 for one sequence of 4097 tokens.
// Other forms, each against this one as it stood then (64 ragged, drafts, shared prefix): eight waves of one kind with the value
// dimensions split 141 / 296 / 234 us against 142 / 260 / 227; four of one kind, one a SIMD, pipelined 142 / 276 / 264.
#include <type_traits>

#include "latent.h"

namespace kda355 {
namespace {

constexpr int SCORE_WAVES = 4;
// Value waves: 4, and 8 from 4 bits with one row tile, where a wave's conversions, one after the other, are the longest way through a step
// (64 ragged sequences of 32 heads: 4 waves 70 us, 8 waves 64).
template <int RT, bool Q4>
constexpr int VALUE_WAVES = Q4 && RT == 1 ? 8 : 4;
template <int RT, bool Q4>
constexpr int THREADS = (SCORE_WAVES + VALUE_WAVES<RT, Q4>) * 64;
constexpr int BN = 32;                                  // keys of a tile
constexpr int MAX_ROWS = 64;                            // query rows of a group
// The cut is by cost: beginning a sequence (lengths, queries, page numbers and first tile one after the other) takes about as
// long as LEAD tiles, which stand in front of every sequence's own; a run is MIN_RUN of these units at least.  Measured: 64
// ragged sequences 138 us with LEAD 4, 134 with 6 and with 8; one sequence of 4097 tokens 14.4 us with runs of 2, 13.9 of 3, 14.3 of 4.
constexpr uint32_t LEAD = 8, MIN_RUN = 3;
// workspace: the cut for the second kernel (run, runs of the prefix), then slots, of 32 rows: accumulators, (m, l) of each row
constexpr int SLOTS = 256, SLOT_ACC = 65536, SLOT_TILE = SLOT_ACC + 256;

__device__ const uint4 zero_rows4[8 * ROW4 / 16] = {};  // what 8 tokens that are not there read, in 4 bits

struct Groups {
    int rows, groups;  // rows of a group, groups
    static Groups of(int64_t n, int most) {
        const int64_t g = (n + most - 1) / most;
        const int64_t r = g ? (n + 32 * g - 1) / (32 * g) * 32 : 32;  // in tiles of 32, about equal
        return {(int)r, (int)((n + r - 1) / r)};
    }
};
struct Plan {
    Groups own, pre;       // of a sequence's rows; of all rows of the batch, for the prefix (no groups: no prefix)
    int grid;
    float per_wg;          // 1 / grid
    int64_t pre_slots;     // workspace: prefix parts, then the sequences' (64 KiB a slot of 32 rows)
    PageOf page;
};

// ------------------------------------------------------------------------------------------------ who does what
struct Cut {
    uint32_t own, pre, run;  // units of all sequences, tiles of the prefix; units of a workgroup
    uint32_t pre_runs, pre_wgs, own_wgs;
};
__device__ __forceinline__ uint32_t tiles_of(int tokens) { return ((uint32_t)tokens + BN - 1) / BN; }
__device__ __forceinline__ uint32_t units_of(int tokens) { return tokens ? tiles_of(tokens) + LEAD : 0; }
__device__ __forceinline__ uint32_t cdiv(uint32_t x, uint32_t y) { return x / y + (x % y != 0); }
// The sequences' tokens: every lane has one of the first 64, loaded once.
struct Lengths {
    const KdaLatentDecodeArgs& a;
    int mine;
    __device__ __forceinline__ int load(int n) const { return tokens_of(a.seq_lens[n], a.table_width, a.page_size); }
    __device__ __forceinline__ explicit Lengths(const KdaLatentDecodeArgs& args) : a(args), mine(load(min((int)(threadIdx.x & 63), args.B - 1))) {}
    __device__ __forceinline__ int of_lane(int n) const { return n >= a.B ? 0 : n < 64 ? mine : load(n); }  // n % 64: the lane
    __device__ __forceinline__ int of(int n) const {  // n: the same in all lanes
        return n < 64 ? __builtin_amdgcn_readlane(mine, n) : __builtin_amdgcn_readfirstlane(load(n));
    }
};

// The shortest run (to 1.6 %) with which the grid covers everything, the same in every wave: the lanes try 64 candidates.
__device__ __forceinline__ Cut cut(const KdaLatentDecodeArgs& a, const Plan& p, uint32_t own) {
    Cut c;
    c.own = own;
    c.pre = p.pre.groups ? tiles_of(tokens_of(a.prefix_len[0], a.prefix_width, a.page_size)) : 0;
    c.pre = __builtin_amdgcn_readfirstlane(c.pre);
    const uint32_t most = max(max(c.own, c.pre), MIN_RUN);  // one run a group: always fits
    const float all = (float)p.pre.groups * (float)c.pre + (float)p.own.groups * (float)c.own, top = (float)most;
    const float lo = fmaxf(fminf(__builtin_ceilf(all * p.per_wg), top), (float)MIN_RUN);
    const int lane = threadIdx.x & 63;
    const float f = lane < 32 ? 1.f + lane * (1.f / 64) : 1.5f * __builtin_amdgcn_exp2f((lane - 31) * 0.25f);
    const uint32_t r = lane == 63 ? most : min((uint32_t)fminf(__builtin_ceilf(lo * f), top), most);
    const uint32_t pre = p.pre.groups ? cdiv(c.pre, r) : 0, mine = cdiv(c.own, r);
    const uint64_t wgs = (uint64_t)p.pre.groups * pre + (uint64_t)p.own.groups * mine;
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(wgs <= (uint32_t)p.grid) | 1ull << 63);
    c.run = __builtin_amdgcn_readlane(r, l);
    c.pre_runs = __builtin_amdgcn_readlane(pre, l);
    c.pre_wgs = p.pre.groups * c.pre_runs;
    c.own_wgs = p.own.groups * __builtin_amdgcn_readlane(mine, l);
    return c;
}
__device__ __forceinline__ uint32_t sum_wave(uint32_t x) { return __builtin_amdgcn_readlane(scan_wave(x), 63); }
struct At { int n; uint32_t before; };
// the sequence that holds unit u of all (u < their sum), and the units before it
__device__ __forceinline__ At sequence_of(const Lengths& lens, uint32_t u) {
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int n0 = 0; n0 < lens.a.B; n0 += 64) {
        const uint32_t t = units_of(lens.of_lane(n0 + lane)), s = scan_wave(t);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(before + s > u);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            return {n0 + l, before + __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(t, l)};
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return {lens.a.B, before};
}

// ------------------------------------------------------------------------------------------------ LDS
// A tile: latent rows in blocks of 4 tokens x 16 pieces of 16 bytes, piece p of token t at block 4 (t / 4) + p / 16, row t % 4,
// place (p % 16) ^ turn(t) (a block is one load of a wave); then the positional parts, piece p of token t at p ^ swz8(t).
// 16-byte reads go 16 lanes at a time, lanes 0 .. 3, 12 .. 15, 20 .. 23, 24 .. 27 of 32 and the others, transposed reads 32 lanes in
// order: with this turn the former touch all 16 places of 256 bytes, and so do the latter.  (A turn that serves the former alone
// and weights without their turn: 35 % more LDS cycles, 1 % more time.)
__device__ __forceinline__ int turn(int t) { return (t & 3) << 2 | (t >> 3 & 1) << 1; }
// From 4 bits 16-byte reads of 16 tokens' same piece (and, by the other lanes, its neighbour p ^ 1) and transposed reads of 8 tokens'
// pieces p and p ^ 1 both touch all 16 places.
__device__ __forceinline__ int turn4(int t) { return ((t & 7) ^ (t & 8) >> 1) << 1 | (t >> 3 & 1); }
// The queries' turn for that order: a lane quarter reads pieces 4 quad .. of 16 rows.
__device__ __forceinline__ int turn_q4(int t) { return (t & 3) << 2 | (t >> 2 & 3); }
constexpr int BLOCK = 1024, LAT_TILE = BN * LAT_BYTES, PE_TILE = BN * PE_BYTES;
template <bool Q4, int VW>
struct Lds {
    // A cache in 16 bits: latent rows and positional parts of four tiles, side by side.  In 4 bits: codes, scales and positional parts of
    // eight tiles as they came, and of every value wave the scales of its values once more, in 32 bits.  A token's 16-byte piece p of
    // codes stands at p ^ turn4(t), its scales at 256 (t / 8) + 16 (t % 8).  The queries come through the first 64 KiB, which the first
    // three tiles of a segment (slots 5 .. 7) leave free.
    static constexpr int THERES = Q4 ? 8 : 4, PAGE_RING = Q4 ? 8 : 4;
    static constexpr int SPREAD = LAT / GROUP / VW * 4;  // bytes a token
    static constexpr int RAW = VW * BN * SPREAD, RAW_SCALES = BN * SCALES4, RAW_PE = RAW_SCALES + 4 * 256, RAW_TILE = RAW_PE + PE_TILE;
    static_assert(RAW + 5 * RAW_TILE >= 2 * LAT_TILE, "");
    static constexpr int P = Q4 ? RAW + 8 * RAW_TILE : 4 * (LAT_TILE + PE_TILE);  // weights: [tile % 2][row tile][16-key step][row][key ^ (row & 8)] 16 bits
    static constexpr int MAX = P + 2 * 4096;             // a tile's maxima [tile % 2][score wave][32], at the end the sums of rows
    static constexpr int FLAG = MAX + 2 * SCORE_WAVES * 128;  // does the wave's tile raise the maximum [tile % 2][score wave]
    static constexpr int THERE = FLAG + 64;              // is the token there [tile % THERES][32] bytes
    static constexpr int PAGES = THERE + THERES * BN;    // page numbers [value wave][tile % PAGE_RING][64]
    static constexpr int BYTES = PAGES + VW * PAGE_RING * 256;
    static constexpr int LOADS = !Q4 ? 10 : VW == 8 ? 3 : 5;  // of a value wave a tile: 8 of latent rows | 2 of codes, scales; positional parts, page numbers
    static_assert(BYTES <= 160 * 1024 && RAW % 1024 == 0 && P % 1024 == 0 && RAW_TILE % 1024 == 0, "");
};

template <int I>
using Int = std::integral_constant<int, I>;
// the four lane groups of 16 joined
template <typename F>
__device__ __forceinline__ float join_groups(float x, F f) {
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = f(__uint_as_float(a.x), __uint_as_float(a.y));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return f(__uint_as_float(b.x), __uint_as_float(b.y));
}

template <typename T, int RT, bool Q4, bool EVEN>
__global__ void __launch_bounds__((THREADS<RT, Q4>), (THREADS<RT, Q4> / 256)) decode_kernel(KdaLatentDecodeArgs a, Plan p) {
    constexpr int VW = VALUE_WAVES<RT, Q4>, DIMS = LAT / VW, DV = DIMS / 32;  // values of a value wave, accumulators of 32
    typedef Lds<Q4, VW> L;
    constexpr int CACHE_ROW = Q4 ? ROW4 : ROW_BYTES;
    __shared__ __align__(1024) unsigned char sm[L::BYTES];
    const uint32_t lds = lds_offset(sm);
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;

    asm volatile("" ::"s"(a.q_latent), "s"(a.ql_row), "s"(a.page_stride), "s"(a.B), "s"(p.grid));  // all arguments at once
    const Lengths lens(a);
    // ---- what does not depend on the lengths, while they come
    const float sc = a.scale * 1.44269504088896f;
    const int64_t page_bytes = Q4 ? a.page_stride : a.page_stride * 2;
    const char* const cache = static_cast<const char*>(a.cache);
    const bool scores = w < SCORE_WAVES;
    const int rw = w & 1, kh = w >> 1 & 1;  // a score wave's rows 16 RT rw .. (16 RT of them) and keys 16 kh ..
    const int vw = w & (VW - 1);            // a value wave's DIMS values (waves SCORE_WAVES .. : in any order)
    const int tw = VW == 8 ? vw >> 1 : vw;  // it brings of tokens 8 tw .. + 7
    // What follows from the lane, from 4 bits anew in every segment: kept, what the waves of one kind read would take the other kind's registers.
    auto my_lane = [&] {
        int l = lane;
        if constexpr (Q4) asm volatile("" : "+v"(l));
        return l;
    };

    uint32_t t0 = 0, t0_ = 0;  // the segment's first tile; the same, unknown to the compiler: addresses of the first tiles would be kept and spilled
    auto lat_at = [&](uint32_t tile) { return lds + tile % 4 * (LAT_TILE + PE_TILE); };            // a tile's latent rows
    auto raw_at = [&](uint32_t tile) { return lds + L::RAW + (tile - t0_ + 5) % 8 * L::RAW_TILE; };  // what came of it in 4 bits
    auto pe_at = [&](uint32_t tile) { return Q4 ? raw_at(tile) + L::RAW_PE : lat_at(tile) + LAT_TILE; };  // its positional parts

    uint32_t own = 0;
    for (int n = lane; n < a.B; n += 64) own += units_of(lens.of_lane(n));
    const Cut cu = cut(a, p, sum_wave(own));
    const uint32_t wgs = cu.pre_wgs + cu.own_wgs;
    if (blockIdx.x == 0 && tid == 0) *static_cast<u32x2*>(a.workspace) = u32x2{cu.run, cu.pre_runs};
    if (blockIdx.x >= wgs) return;
    const uint32_t task = xcd_task(blockIdx.x, wgs);  // neighbours read the same keys: on one XCD
    const bool prefix = task < cu.pre_wgs;
    const Groups gr = prefix ? p.pre : p.own;
    const uint32_t id = __builtin_amdgcn_readfirstlane(prefix ? task : task - cu.pre_wgs);
    const uint32_t piece = __builtin_amdgcn_readfirstlane(id / gr.groups);
    const int g = __builtin_amdgcn_readfirstlane(id - piece * gr.groups);
    const uint32_t end = min((piece + 1) * cu.run, prefix ? cu.pre : cu.own);
    uint32_t u = piece * cu.run;
    At at = {0, 0};
    if (!prefix) at = sequence_of(lens, u);

    while (u < end) {
        // ---- the segment: key tiles [t0, t1) of one key sequence, for rows [r0, r1) of the batch
        int n = 0, tokens, r0, r1;
        uint32_t t1, whole;
        const int32_t* table;
        int width;
        if (prefix) {
            tokens = tokens_of(a.prefix_len[0], a.prefix_width, a.page_size);
            table = a.prefix_table, width = a.prefix_width;
            r0 = g * gr.rows, r1 = min(r0 + gr.rows, a.B * a.S * a.H);
            t0 = u, t1 = end, whole = 0;
            u = end;
        } else {
            n = at.n;
            tokens = lens.of(n);
            table = a.block_table + n * a.table_stride, width = a.table_width;
            const int rows = a.S * a.H;
            r0 = n * rows + g * gr.rows, r1 = min(r0 + gr.rows, (n + 1) * rows);
            const uint32_t tiles = tiles_of(tokens), units = units_of(tokens);
            const uint32_t from = u - at.before, to = min(units, end - at.before);
            t0 = from > LEAD ? from - LEAD : 0, t1 = to > LEAD ? to - LEAD : 0;
            whole = t0 == 0 && t1 == tiles && cu.pre == 0;
            u = at.before + to;
            if (to == units) at = {n + 1, at.before + units};
        }
        tokens = __builtin_amdgcn_readfirstlane(tokens);
        if (t0 >= t1) continue;  // no tokens, or not the first
        // tokens that a row sees: all for the prefix, all but the draft tokens after its own for a sequence
        const int hidden = prefix ? 0 : a.S - 1 + n * a.S;  // (minus the row's token)
        auto sees = [&](int r) { return prefix ? tokens : tokens - (hidden - r / a.H); };
        const int first = __builtin_amdgcn_readfirstlane(sees(r0)), last = __builtin_amdgcn_readfirstlane(sees(r1 - 1));
        const uint32_t stop = max(t0, min(t1, last > 0 ? ((uint32_t)last + BN - 1) / BN : 0u));

        const uint32_t n_tiles = stop - t0;
        t0_ = __builtin_amdgcn_readfirstlane(t0);
        asm volatile("" : "+s"(t0_));
        // A tile's weights are relative to a past maximum of their rows, which is raised only when some row of a wave exceeds it
        // by SLACK (the result is the same for any reference): after the fact, at the start of the next step.
        auto flags = [&](uint32_t tile) { return *reinterpret_cast<const u32x4*>(sm + L::FLAG + (tile & 1) * 16); };
        auto any = [](u32x4 fl) { return __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0; };
        // the new reference of the group's row r after `tile`, by its own scores alone; returns the factor of what is there
        auto raise = [&](uint32_t tile, int r, float& m) {
            const float m0 = *reinterpret_cast<const float*>(sm + L::MAX + (tile & 1) * 512 + r * 4);
            const float m1 = *reinterpret_cast<const float*>(sm + L::MAX + (tile & 1) * 512 + (MAX_ROWS + r) * 4);
            const float mx = fmaxf(m0, m1), mn = mx - m > T::B + T::SLACK ? mx - T::B : m, f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            return f;
        };
        if (scores) {
            // ================================================================ score waves
            const int my = my_lane(), c16 = my & 15, quad = my >> 4, c = my & 31;
            // LDS read addresses within a tile: key 16 kh + c16, dimensions 8 quad .. of a 32-dimension step, latent and positional
            const int key_at = 16 * kh + c16;
            const uint32_t ra[2] = {(uint32_t)(Q4 ? key_at * SCALES4 + ((quad ^ turn4(c16)) << 4)
                                                  : (key_at >> 2) * (4 * BLOCK) + (key_at & 3) * 256 + ((quad ^ turn(key_at)) << 4)),
                                    (uint32_t)(key_at * PE_BYTES + ((quad ^ swz8(key_at)) << 4))};
            const int row0 = r0 + 16 * RT * rw + c16;  // this lane's rows: row0, and with two row tiles row0 + 16
            // The queries come through the LDS of tiles t0 + 2 and t0 + 3 (from 4 bits: the first 64 KiB and the weights'), a row tile in each, laid out like keys, half of a wave's
            // rows by it and half by the other wave that has them (rows past the end repeat the last one).  (Straight into registers,
            // 64 bytes of 16 rows at a time and every row twice, 4900 cycles until the first tile was there, and 10800 in 64 sequences of
            // 64 heads; 1900 and 4800 so.)
            int mine[RT];
            const uint32_t qx = RT > 1 ? rw : 0, qb = Q4 ? lds + qx * LAT_TILE : lat_at(t0 + 2 + qx);
            const uint32_t qpe = Q4 ? lds + L::P + qx * PE_TILE : pe_at(t0 + 2 + qx);
            const bool some = n_tiles && row0 - c16 < r1;
            auto half_of = [&](int x) { return RT > 1 ? x : rw; };  // of the row tile: where rows row0 + 16 x stand
            {
                int me = lane;  // (not kept from one segment to the next: there are no registers for it)
                asm volatile("" : "+v"(me));
                const int x0 = RT > 1 ? kh : 0, at0 = RT > 1 ? 0 : 8 * kh;  // this wave loads rows row0 - c16 + 16 x0 + at0 ..
                uint64_t latent = 0, pe = 0;                                // of row row0 + 16 x0
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    const int r = min(row0 + 16 * x, r1 - 1), t = r / a.H, h = r - t * a.H;
                    mine[x] = sees(r);
                    if (x == x0) {
                        latent = (uint64_t)(static_cast<const uint16_t*>(a.q_latent) + t * a.ql_row + h * a.ql_head);
                        pe = (uint64_t)(static_cast<const uint16_t*>(a.q_pe) + t * a.qp_row + h * a.qp_head);
                    }
                }
                if (some) {
                    const uint32_t block = qb + (4 * half_of(x0) + at0 / 4) * (4 * BLOCK);
                    const uint32_t pe_block = qpe + (16 * half_of(x0) + at0) * PE_BYTES;
#pragma unroll
                    for (int i = 0; i < 2 * RT; ++i) {
                        const int t = at0 + 4 * i + (me >> 4);
                        const uint64_t from = of_lane(latent, t) + (((me & 15) ^ (Q4 ? turn_q4(t) : turn(t))) << 4);
                        const uint32_t to = block + i * (4 * BLOCK);
                        load_block<0>(to, from);
                        load_block<256>(to + BLOCK, from);
                        load_block<512>(to + 2 * BLOCK, from);
                        load_block<768>(to + 3 * BLOCK, from);
                    }
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        const int t = at0 + 8 * i + (me >> 3);
                        load_block<0>(pe_block + 8 * i * PE_BYTES, of_lane(pe, t) + (((me & 7) ^ swz8(t)) << 4));
                    }
                }
            }
            wait_loads<0>();
            lds_barrier();  // the first tile, the queries
            u32x4 q[RT][18] = {};
            if (some) {
                int me = lane;
                asm volatile("" : "+v"(me));
                const int c16 = me & 15, quad = me >> 4;
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    // Step i of the scores takes values 32 i + 8 quad .., from 4 bits, where a lane reads all 32 of a scale, 128 (i / 4) +
                    // 32 quad + 8 (i % 4) .. (the order of the contraction is free).
                    const int row = 16 * half_of(x) + c16;
                    const uint32_t at4 = qb + (row >> 2) * (4 * BLOCK) + (row & 3) * 256 + ((quad << 2 ^ turn_q4(row)) << 4);
                    const uint32_t at = qb + (row >> 2) * (4 * BLOCK) + (row & 3) * 256 + ((quad ^ turn(row)) << 4), pat = qpe + row * PE_BYTES + ((quad ^ swz8(row)) << 4);
#pragma unroll
                    for (int i = 0; i < 16; ++i) q[x][i] = lds_read16((Q4 ? at4 ^ ((i & 3) << 4) : at ^ ((i & 3) << 6)) + (i >> 2) * BLOCK);
#pragma unroll
                    for (int i = 0; i < 2; ++i) q[x][16 + i] = lds_read16(pat ^ (i << 6));
                }
            }
            lds_barrier();  // the queries are in registers
            float mo[RT], l[RT] = {}, sum[RT] = {};
#pragma unroll
            for (int x = 0; x < RT; ++x) mo[x] = M_START;
            f32x4 s[RT] = {};
            auto weights = [&](uint32_t tile, int x) {  // of rows row0 + 16 x, relative to mo[x]; leaves their sum
                float p0[4];
                sum[x] = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p0[r] = __builtin_amdgcn_exp2f(fmaf(s[x][r], sc, -mo[x]));
                    sum[x] += p0[r];
                }
                *reinterpret_cast<u32x2*>(sm + L::P + (tile & 1) * 4096 + (2 * (RT > 1 ? rw : 0) + kh) * 1024 + half_of(x) * 512 + c16 * 32 +
                                          (quad ^ (c16 >> 3) << 1) * 8) =
                    u32x2{T::pack(p0[0], p0[1]), T::pack(p0[2], p0[3])};
            };
            auto settle = [&](uint32_t tile, u32x4 fl) {  // what the step of `tile` left open
                if (any(fl)) {
                    if (RT == 1 || __builtin_amdgcn_readfirstlane(rw ? fl[1] | fl[3] : fl[0] | fl[2]))
#pragma unroll
                        for (int x = 0; x < RT; ++x) {
                            l[x] *= raise(tile, 16 * RT * rw + 16 * x + c16, mo[x]);
                            weights(tile, x);
                        }
                    lds_barrier();  // the weights anew
                }
#pragma unroll
                for (int x = 0; x < RT; ++x) l[x] += sum[x];
            };
            u32x4 fl = {};
            // from 4 bits: the lane's part of its key, read a tile ahead
            u32x4 codes[4], scales, pe[2];
            auto fetch = [&](uint32_t tile) {
                const uint32_t tb = raw_at(tile);
#pragma unroll
                for (int j = 0; j < 4; ++j) codes[j] = lds_read16((tb + ra[0]) ^ (j << 6));
                scales = lds_read16(tb + L::RAW_SCALES + (2 * kh + (c16 >> 3)) * 256 + (c16 & 7) * 16);
#pragma unroll
                for (int i = 0; i < 2; ++i) pe[i] = lds_read16((tb + L::RAW_PE + ra[1]) ^ (i << 6));
            };
            if (Q4 && n_tiles) fetch(t0);
            for (uint32_t tile = t0; tile < stop; ++tile) {
                const uint32_t tb = lat_at(tile), tp = pe_at(tile);
                const int k0 = (int)(tile * BN);
                if (tile > t0) fl = flags(tile - 1);
                const int there8 = *(sm + L::THERE + (tile % L::THERES) * BN + c);
                // ---- 18 steps for both halves of the rows, in two chains each, the operands read five steps ahead
                auto key = [&](int i) {
                    return i < 16 ? lds_read16(((tb + ra[0]) ^ ((i & 3) << 6)) + (i >> 2) * BLOCK) : lds_read16((tp + ra[1]) ^ ((i - 16) << 6));
                };
                f32x4 z[RT][2] = {};
                if constexpr (Q4) {
                    settle(tile - 1, fl);
                    auto key4 = [&](int i) {  // (the exponent in place: the conversion looks at nothing else of the scale)
                        const uint32_t s4 = scales[i >> 2 & 3];
                        return i < 16 ? T::from4(codes[i >> 2 & 3][i & 3], __uint_as_float(__builtin_amdgcn_alignbit(s4, s4, 8 * quad + 9))) : pe[i & 1];
                    };
                    u32x4 kf[2] = {key4(0)};
#pragma unroll
                    for (int i = 0; i < 18; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (i + 1 < 18) kf[(i + 1) & 1] = key4(i + 1);
#pragma unroll
                        for (int y = 0; y < RT; ++y) z[y][i & 1] = T::mfma16(kf[i & 1], q[y][i], z[y][i & 1]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(tile + 1);
                } else {
                    u32x4 kf[6];
#pragma unroll
                    for (int i = 0; i < 5; ++i) kf[i] = key(i);
                    __builtin_amdgcn_sched_barrier(0);
                    settle(tile - 1, fl);
#pragma unroll
                    for (int i = 0; i < 18; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (i + 5 < 18) kf[(i + 5) % 6] = key(i + 5);
#pragma unroll
                        for (int y = 0; y < RT; ++y) z[y][i & 1] = T::mfma16(kf[i % 6], q[y][i], z[y][i & 1]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < RT; ++x) s[x] = z[x][0] + z[x][1];
                const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(there8 != 0);
                if (k0 + BN > first || there != ~0u) {
#pragma unroll
                    for (int x = 0; x < RT; ++x) {
                        const int left = mine[x] - k0;
                        const uint32_t vis = (there & (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u)) >> (16 * kh + 4 * quad);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!(vis >> r & 1)) s[x][r] = -INFINITY;
                    }
                }
                float mx[RT];
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    mx[x] = fmaxf(fmaxf(s[x][0], s[x][1]), fmaxf(s[x][2], s[x][3]));
                    mx[x] = join_groups(mx[x], [](float p, float q) { return fmaxf(p, q); }) * sc;
                    *reinterpret_cast<float*>(sm + L::MAX + (tile & 1) * 512 + (MAX_ROWS * kh + 16 * RT * rw + 16 * x + c16) * 4) = mx[x];  // (the groups' values agree)
                    weights(tile, x);
                }
                const bool up = __builtin_amdgcn_ballot_w64(fmaxf(mx[0] - mo[0], mx[RT - 1] - mo[RT - 1]) > T::B + T::SLACK) != 0;
                *reinterpret_cast<int*>(sm + L::FLAG + (tile & 1) * 16 + w * 4) = up;
                lds_barrier();  // the tile's weights; the next tile is whole
            }
            if (n_tiles) settle(stop - 1, flags(stop - 1));
            lds_barrier();  // the last maxima are read
#pragma unroll
            for (int x = 0; x < RT; ++x) {
                l[x] = join_groups(l[x], [](float p, float q) { return p + q; });
                if (quad == 0) *reinterpret_cast<float*>(sm + L::MAX + (MAX_ROWS * kh + 16 * RT * rw + 16 * x + c16) * 4) = l[x];
            }
            lds_barrier();
            lds_barrier();  // the value waves have read it
            continue;
        }

        // ==================================================================== value waves
        const int my = my_lane(), c16 = my & 15, quad = my >> 4, c = my & 31, half = my >> 5;
        // LDS read addresses within a tile: values as operand rows (key 8 half + e of a 16-key step is element e), e < 4 and from 4 on
        uint32_t ra[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int t = 8 * half + 4 * x + (c16 >> 2);
            const int e = 2 * (quad & 1) + ((c16 & 3) >> 1);
            ra[x] = (t >> 2) * (4 * BLOCK) + (t & 3) * 256 + vw * BLOCK + ((e ^ turn(t)) << 4) + (c16 & 1) * 8;
        }
        // ---- loads
        const uint32_t pages = (uint32_t)min(a.pages, (int64_t)1 << 31);
        const u32x4 table_rsrc = tile_rsrc(table, (uint32_t)width * 4);  // entries past the table read as zeros (and are past `last`)
        const uint32_t pages_at = lds + L::PAGES + vw * (L::PAGE_RING * 256);
        int me = lane;  // (computed anew for every segment: the score waves have no registers for what follows from it)
        asm volatile("" : "+v"(me));
        const int own8 = 8 * tw + (me & 7);  // this lane finds the address of one token
        auto load_pages = [&](uint32_t tile) {  // the page numbers of the wave's tokens
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(
                             __builtin_amdgcn_readfirstlane(pages_at + tile % L::PAGE_RING * 256)),
                         "v"(p.page(tile * BN + own8) * 4), "s"(table_rsrc)
                         : "memory");
        };
        // where the next tile to be brought stands: this lane's pieces of 4 + 4 tokens and of the positional parts, found in
        // steps that can be spread: the page, the address of the lane's token, the addresses for the lane's pieces
        uint64_t at_latent[2], at_pe, at_scales;
        auto find_page = [&](uint32_t tile) {
            return *(__attribute__((address_space(3))) const int*)(lds_byte*)(uintptr_t)(pages_at + tile % L::PAGE_RING * 256 + (EVEN ? 0 : my * 4));
        };
        // EVEN: the wave's 8 tokens stand in one page in a row, so one address and fixed offsets lead to all of them.  (Tokens past the
        // last are read as they are: no row sees them.  spread_scales takes their values out.)
        auto find_rows = [&](uint32_t tile, int page) {
            const uint32_t tok = tile * BN + 8 * tw, pg = __builtin_amdgcn_readfirstlane(page);
            const bool there = tok < (uint32_t)last && pg < pages;
            *(sm + L::THERE + (tile % L::THERES) * BN + own8) = there && tile * BN + own8 < (uint32_t)last;
            const uint64_t at = (uint64_t)cache + pg * (uint64_t)page_bytes + (uint64_t)(tok - p.page(tok) * (uint32_t)a.page_size) * CACHE_ROW;
            return there ? at : (uint64_t)zero_rows4;
        };
        auto find_token = [&](uint32_t tile, int page) {
            const uint32_t tok = tile * BN + own8;
            const bool in = tok < (uint32_t)last && (uint32_t)page < pages;  // in the tokens that the group sees, no hole
            *(sm + L::THERE + (tile % L::THERES) * BN + own8) = in;
            uint64_t at = (uint64_t)cache + (uint32_t)page * (uint64_t)page_bytes +
                          (uint64_t)(tok - p.page(tok) * (uint32_t)a.page_size) * CACHE_ROW;
            asm volatile("" : "+v"(at));  // (a choice of two, not a branch)
            return in ? at : (uint64_t)zero_row;
        };
        auto place = [&](int t) { return (uint32_t)((me & 15) ^ (Q4 ? turn4(t & 15) : turn(t))) << 4; };
        const int four = VW == 8 ? vw & 1 : 0;  // with 8 value waves: of the 8 tokens the 4 whose codes the wave brings; beside them scales or positional parts
        const uint32_t piece4[2] = {place(8 * tw + 4 * four + (me >> 4)), place(8 * tw + 4 + (me >> 4))};
        const uint32_t piece8 = (Q4 ? PE4 : LAT_BYTES) + (((me & 7) ^ swz8(8 * tw + (me >> 3))) << 4);
        auto find_latent = [&](uint64_t at, int x) { at_latent[x] = of_lane(at, 4 * (x + four) + (me >> 4)) + piece4[x]; };
        auto find_pe = [&](uint64_t at) { at_pe = of_lane(at, me >> 3) + piece8; };
        const uint32_t off4[4] = {(uint32_t)(4 * four + (me >> 4)) * ROW4 + piece4[0], (uint32_t)(4 + (me >> 4)) * ROW4 + piece4[1],
                                  (uint32_t)(me >> 2 & 7) * ROW4 + SCALES4 + (me & 3) * 4, (uint32_t)(me >> 3) * ROW4 + piece8};
        auto bring_even = [&](uint32_t tile, uint64_t at, int i) {
            if (i == 0 || (i == 1 && VW == 4)) load_block_from(raw_at(tile) + (2 * tw + four + i) * BLOCK, at, off4[i]);
            if (i == 2 && !four) load_words_from(raw_at(tile) + L::RAW_SCALES + tw * 256, at, off4[2]);
            if (i == 3 && (VW == 4 || four)) load_block_from(pe_at(tile) + 8 * tw * PE_BYTES, at, off4[3]);
        };
        auto find_scales = [&](uint64_t at) { at_scales = of_lane(at, me >> 2 & 7) + (SCALES4 + (me & 3) * 4); };
        auto bring = [&](uint32_t tile, auto i) {  // load i of 9: four of 4 tokens, four of 4 more, the positional parts
            constexpr int I = decltype(i)::value;
            if constexpr (I == 8) {
                if (VW == 4 || four) load_block<0>(pe_at(tile) + 8 * tw * PE_BYTES, at_pe);
            } else if constexpr (!Q4)
                load_block<(I & 3) * 256>(lat_at(tile) + (2 * vw + (I >> 2)) * (4 * BLOCK) + (I & 3) * BLOCK, at_latent[I >> 2]);
            else if constexpr (I == 0 || (I == 1 && VW == 4))
                load_block<0>(raw_at(tile) + (2 * tw + four + I) * BLOCK, at_latent[I]);  // of 4 bits: codes of 4 tokens and of 4 more, the scales
            else if constexpr (I == 2) {
                if (!four) load_words(raw_at(tile) + L::RAW_SCALES + tw * 256, at_scales);
            }
        };
        // [row tile][32 values]: from 16 bits values 32 d + i, from 4 bits 64 (d / 2) + 2 i + d % 2, i = (e & 3) + 8 (e >> 2) + 4 half
        f32x16 acc[RT][DV] = {};
        float mo[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) mo[r] = M_START;
        bool special = false;
        // One step: `tile` added, the value waves' loads of tile + AHEAD (past the end: zeros) and the addresses of the one after
        // it between the products.  LAST: nothing is brought.
        constexpr uint32_t AHEAD = 3;
        auto step = [&](uint32_t tile, auto last_) {
            constexpr bool LAST = decltype(last_)::value;
            const bool mixed = (int)(tile * BN + BN) > first;  // some row does not see some token of the tile
            const uint32_t vb = lat_at(tile), pb = lds + L::P + (tile & 1) * 4096 + c * 32 + (half ^ (c >> 3 & 1)) * 16;
            auto value = [&](int k, int d) {
                const u32x2 v0 = lds_read_tr(((vb + ra[0]) ^ (d << 6)) + k * 16 * BLOCK);
                const u32x2 v1 = lds_read_tr(((vb + ra[1]) ^ (d << 6)) + k * 16 * BLOCK);
                return u32x4{v0.x, v0.y, v1.x, v1.y};
            };
            auto weight = [&](int k, int r) { return lds_read16(pb + (2 * r + k) * 1024); };
            const u32x4 fl = flags(tile);
            u32x4 vf[4], pf[RT];
            int page = 0;
#pragma unroll
            for (int r = 0; r < RT; ++r) pf[r] = weight(0, r);
#pragma unroll
            for (int d = 0; d < 4; ++d) vf[d] = value(0, d);
            if constexpr (!LAST) page = find_page(tile + AHEAD + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (any(fl)) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (RT > 1 && !__builtin_amdgcn_readfirstlane(fl[r] | fl[r + 2])) continue;
                    const float f = raise(tile, 32 * r + c, mo[r]);
                    if (tile != t0)  // (nothing is there yet)
#pragma unroll
                        for (int d = 0; d < 4; ++d) acc[r][d] *= f;
                }
                lds_barrier();  // the weights anew
#pragma unroll
                for (int r = 0; r < RT; ++r) pf[r] = weight(0, r);
            }
            uint64_t at = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                u32x4 pn[RT];
                if (mixed)
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        special |= nonfinite<T>(vf[d]);
                        vf[d] = finite_part<T>(vf[d]);
                    }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r][d] = T::mfma(vf[d], pf[r], acc[r][d]);
                    if (k == 0) {  // the second half's operands
                        vf[d] = value(1, d);
                        if (d == 2)
#pragma unroll
                            for (int r = 0; r < RT; ++r) pn[r] = weight(1, r);
                    }
                    if constexpr (!LAST) {  // (what an address is taken from is needed no more)
                        if (k == 0) {
                            if (d == 0) bring(tile + 3, Int<0>{});
                            if (d == 1) bring(tile + 3, Int<1>{}), at = find_token(tile + 4, page);
                            if (d == 2) bring(tile + 3, Int<2>{});
                            if (d == 3) bring(tile + 3, Int<3>{}), bring(tile + 3, Int<8>{});
                        } else {
                            if (d == 0) bring(tile + 3, Int<4>{}), find_latent(at, 0);
                            if (d == 1) bring(tile + 3, Int<5>{}), find_pe(at);
                            if (d == 2) bring(tile + 3, Int<6>{}), load_pages(tile + 6);
                            if (d == 3) bring(tile + 3, Int<7>{}), find_latent(at, 1);
                        }
                    }
                }
                if (k == 0)
#pragma unroll
                    for (int r = 0; r < RT; ++r) pf[r] = pn[r];
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!LAST) {
                wait_loads<L::LOADS>();
                lds_barrier();  // the next tile's weights; the tile after it is whole
            }
        };
        // The same from 4 bits.  A transposed read of bytes gives a lane 8 tokens' codes of values 2 m and 2 m + 1 (m = l % 32 of 64 values):
        // eight conversions and eight exchanges of halves make one operand of even values and one of odd ones.  The scales the wave writes out
        // first, as the conversion takes them (64 ragged sequences of 32 heads 62.5 us with the join; 65.3 with 7 shifts for 8 bytes of a transposed read).  A
        // step multiplies what the step before made and makes the next tile's, so that no read of LDS is waited for but the weights'.
        const int tk = 8 * half + (c16 >> 1), pc = quad & 1;  // of 16 tokens the one whose bytes this lane reads; of two pieces the one
        const uint32_t at_codes = tk * SCALES4 + (((DV * vw + pc) ^ turn4(tk)) << 4) + (c16 & 1) * 8;
        constexpr int NB = DV / 2, G = 2 * NB;  // blocks of 64 values, groups of a tile: [16 tokens][64 values]
        const uint32_t spread = lds + vw * (BN * L::SPREAD), at_spread = spread + pc * (BN * 4) + half * 32;  // [32 values][token]
        // lane l spreads the scales of token l / 2: with 4 value waves two of the wave's four, with 8 one of two
        const uint32_t at_scale = L::RAW_SCALES + (my >> 4) * 256 + (my >> 1 & 7) * 16 + DV * vw + (my & 1) * NB;
        u32x4 vf[G][2];  // [group][even, odd]
        uint32_t scale;
        u32x2 code[G];
        auto read_codes = [&](uint32_t tile) {
            const uint32_t from = raw_at(tile);
            if constexpr (NB == 2)
                scale = *(__attribute__((address_space(3))) const uint16_t*)(lds_byte*)(uintptr_t)(from + at_scale);
            else
                scale = *(__attribute__((address_space(3))) const uint8_t*)(lds_byte*)(uintptr_t)(from + at_scale);
#pragma unroll
            for (int g = 0; g < G; ++g) code[g] = lds_read_tr8(((from + at_codes) ^ (g % NB) << 5) + g / NB * (16 * SCALES4));
        };
        u32x4 scales[2][2];  // of 8 tokens, for two groups
        // Of a page's places behind the tokens nobody knows what they hold, and in EVEN they come as they stand: scaled by 2^-127 they are
        // finite, so that no walk for values that are not follows from them (one sequence of 4127 tokens, 12 heads: 14.3 us; 62 with the walk).
        // Only a segment's last tile can have some: ENDS where it may be that one.  (In every step: drafts 234 us for 227.)
        auto spread_scales = [&](uint32_t tile, auto ends) {
            if (EVEN && decltype(ends)::value && (int)(tile * BN) + (my >> 1) >= last) scale = 0;
            auto* to = (__attribute__((address_space(3))) uint32_t*)(lds_byte*)(uintptr_t)(spread + (my & 1) * (NB * BN * 4) + (my >> 1) * 4);
            to[0] = scale << 23;
            if (NB == 2) to[BN] = (scale & 0xff00u) << 15;
            asm volatile("" ::: "memory");
        };
        auto read_scales = [&](int g) {
#pragma unroll
            for (int i = 0; i < 2; ++i) scales[g & 1][i] = lds_read16(at_spread + g % NB * (2 * BN * 4) + g / NB * 64 + i * 16);
        };
        auto widen = [&](int g, bool mixed) {
            uint32_t x[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t c4 = code[g][i];
                const u32x4 s4 = scales[g & 1][i];
                x[4 * i] = T::template pair4<0>(c4, __uint_as_float(s4[0]));
                x[4 * i + 1] = T::template pair4<1>(c4, __uint_as_float(s4[1]));
                x[4 * i + 2] = T::template pair4<2>(c4, __uint_as_float(s4[2]));
                x[4 * i + 3] = T::template pair4<3>(c4, __uint_as_float(s4[3]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                vf[g][0][j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
                vf[g][1][j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
            }
            if (mixed)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    special |= nonfinite<T>(vf[g][i]);
                    vf[g][i] = finite_part<T>(vf[g][i]);
                }
        };
        auto is_mixed = [&](uint32_t tile) { return (int)(tile * BN + BN) > first; };  // some row does not see some token of the tile
        constexpr uint32_t AHEAD4 = 7;
        // the loads of all tiles up to `tile` have arrived, if those of tiles up to `issued` were the last
        auto wait_tile = [&](uint32_t tile, uint32_t issued) {
            const uint32_t left = tile < issued ? issued - tile : 0;
            if (left == 0) wait_loads<0>();
            else if (left == 1) wait_loads<L::LOADS>();
            else if (left == 2) wait_loads<2 * L::LOADS>();
            else if (left == 3) wait_loads<3 * L::LOADS>();
            else wait_loads<4 * L::LOADS>();
        };
        auto step4 = [&](uint32_t tile, auto kind) {  // 0: with loads, 1: none are left, 2: the last one
            constexpr bool LAST = decltype(kind)::value == 2, BRINGS = decltype(kind)::value == 0;  // (then AHEAD4 tiles or more follow this one)
            const uint32_t pb = lds + L::P + (tile & 1) * 4096 + c * 32 + (half ^ (c >> 3 & 1)) * 16;
            auto weight = [&](int k, int r) { return lds_read16(pb + (2 * r + k) * 1024); };
            const u32x4 fl = flags(tile);
            u32x4 pf[2][RT];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int r = 0; r < RT; ++r) pf[k][r] = weight(k, r);
            int page = 0;
            if constexpr (!LAST) {
                if constexpr (BRINGS) page = find_page(tile + AHEAD4);
                read_codes(tile + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (any(fl)) {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (RT > 1 && !__builtin_amdgcn_readfirstlane(fl[r] | fl[r + 2])) continue;
                    const float f = raise(tile, 32 * r + c, mo[r]);
                    if (tile != t0)  // (nothing is there yet)
#pragma unroll
                        for (int d = 0; d < DV; ++d) acc[r][d] *= f;
                }
                lds_barrier();  // the weights anew
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int r = 0; r < RT; ++r) pf[k][r] = weight(k, r);
            }
            const bool mixed = is_mixed(tile + 1);
            uint64_t at = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r][2 * (g % NB) + i] = T::mfma(vf[g][i], pf[g / NB][r], acc[r][2 * (g % NB) + i]);
                if constexpr (!LAST) {
                    if (g == 0) spread_scales(tile + 1, std::bool_constant<!BRINGS>{});
                    read_scales(g);
                    if constexpr (BRINGS && EVEN) {
                        if (g == 0) at = find_rows(tile + AHEAD4, page);
                        if (g == 1) bring_even(tile + AHEAD4, at, 0);
                        if (g == G / 2) bring_even(tile + AHEAD4, at, 1), bring_even(tile + AHEAD4, at, 2);
                        if (g == G - 1) bring_even(tile + AHEAD4, at, 3);
                    } else if constexpr (BRINGS) {
                        if (g == 0) at = find_token(tile + AHEAD4, page), find_latent(at, 0), find_latent(at, 1);
                        if (g == 1) bring(tile + AHEAD4, Int<0>{}), find_scales(at), find_pe(at);
                        if (g == G / 2) bring(tile + AHEAD4, Int<1>{});
                        if (g == G - 1) bring(tile + AHEAD4, Int<2>{}), bring(tile + AHEAD4, Int<8>{});
                    }
                    if (BRINGS && g == G - 1) load_pages(tile + AHEAD4 + 8);
                    if (g > 0) widen(g - 1, mixed);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!LAST) {
                widen(G - 1, mixed);
                if constexpr (BRINGS) wait_loads<4 * L::LOADS>(); else wait_tile(tile + 3, stop - 1);
                lds_barrier();  // the next tile's weights; the two tiles after it are whole
            }
        };
        if (n_tiles) {
#pragma unroll
            for (int i = 0; i < L::PAGE_RING; ++i) load_pages(t0 + i);
            wait_loads<0>();
            auto find_tile = [&](uint32_t tile) {
                const uint64_t at = find_token(tile, find_page(tile));
                find_latent(at, 0), find_latent(at, 1), find_pe(at);
                if constexpr (Q4) find_scales(at);
            };
            auto bring_tile = [&](uint32_t tile) {
                bring(tile, Int<0>{}), bring(tile, Int<1>{}), bring(tile, Int<2>{}), bring(tile, Int<3>{}), bring(tile, Int<4>{});
                bring(tile, Int<5>{}), bring(tile, Int<6>{}), bring(tile, Int<7>{}), bring(tile, Int<8>{});
                if constexpr (Q4) load_pages(tile + L::PAGE_RING);
            };
            auto whole_tile = [&](uint32_t tile) {
                if constexpr (EVEN) {
                    const uint64_t at = find_rows(tile, find_page(tile));
#pragma unroll
                    for (int i = 0; i < 4; ++i) bring_even(tile, at, i);
                    load_pages(tile + L::PAGE_RING);
                    return;
                }
                find_tile(tile);
                bring_tile(tile);
            };
            if constexpr (Q4) {
                // Tiles past the end are not brought (64 ragged sequences of 32 heads 60.6 us, 62.6 with them; one sequence 14.6, 15.2).
                const uint32_t end = stop - 1;
                auto some_tile = [&](uint32_t tile) {
                    if (tile <= end) whole_tile(tile);
                };
                whole_tile(t0);
                some_tile(t0 + 1);
                some_tile(t0 + 2);
                wait_tile(t0, min(t0 + 2, end));
                lds_barrier();  // the first tile, the queries
                wait_tile(t0 + 1, min(t0 + 2, end));
                lds_barrier();  // the queries are in registers; the second tile
                // while the first tile's scores are computed: its values, and tiles t0 + 3 and on
                read_codes(t0);
                spread_scales(t0, std::true_type{});
#pragma unroll 1
                for (uint32_t i = 3; i < AHEAD4; ++i) some_tile(t0 + i);
#pragma unroll
                for (int g = 0; g < G; ++g) read_scales(g), widen(g, is_mixed(t0));
                wait_tile(t0 + 2, min(t0 + AHEAD4 - 1, end));
                lds_barrier();  // the first tile's weights; the second tile is whole
                uint32_t tile = t0;
                for (; tile + AHEAD4 < stop; ++tile) step4(tile, Int<0>{});
                for (; tile < end; ++tile) step4(tile, Int<1>{});
                step4(tile, Int<2>{});
            } else {
                whole_tile(t0);
                whole_tile(t0 + 1);
                load_pages(t0 + 4);
                wait_loads<L::LOADS>();
                lds_barrier();  // the first tile, the queries
                lds_barrier();  // the queries are in registers
                // while the first tile's scores are computed: tile t0 + 2, and where t0 + 3 stands
                whole_tile(t0 + 2);
                find_tile(t0 + 3);
                load_pages(t0 + 5);
                wait_loads<L::LOADS>();
                lds_barrier();  // the first tile's weights; the second tile is whole
                for (uint32_t tile = t0; tile + 1 < stop; ++tile) step(tile, std::false_type{});
                step(stop - 1, std::true_type{});
            }
            wait_loads<0>();  // what was brought past the end
        } else {
            lds_barrier();
            lds_barrier();
        }

        // Infinite or NaN values in tiles that not every row sees whole (from the tile of `first` on).  A row that sees such a token has a
        // score of +inf or NaN, and NaN throughout, or one of -inf, and with it a weight of 0 and a NaN in place of this value.
        if (__builtin_amdgcn_ballot_w64(special)) {
#pragma unroll 1
            for (int j = max(first & ~(BN - 1), (int)(t0 * BN)); j < min(last, (int)(stop * BN)); ++j) {
                const int page = table[j / a.page_size];
                if (page < 0 || page >= a.pages) continue;
                const char* row = cache + page * page_bytes + (int64_t)(j % a.page_size) * CACHE_ROW;
                int my = half;  // (addresses found here: kept from before the loops they would take their registers)
                asm volatile("" : "+v"(my));
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int i = r0 + 32 * r + c;
                    const bool seen = i < r1 && j < sees(min(i, r1 - 1));
                    auto give = [&](float& x, uint32_t value) {
                        if (seen && !(fabsf(T::up((uint16_t)value)) < INFINITY)) x = NAN;
                    };
                    if constexpr (Q4) {
#pragma unroll
                        for (int d = 0; d < DV / 2; ++d)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {  // 8 values in a row
                                const int at = DIMS * vw + 64 * d + 16 * e + 8 * my;
                                const uint32_t b = *reinterpret_cast<const uint8_t*>(row + SCALES4 + at / GROUP);
                                const u32x4 x = T::from4(*reinterpret_cast<const uint32_t*>(row + at / 2), __uint_as_float(b << 23));
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    float even = acc[r][2 * d][4 * e + k], odd = acc[r][2 * d + 1][4 * e + k];
                                    give(even, x[k]), give(odd, x[k] >> 16);
                                    acc[r][2 * d][4 * e + k] = even, acc[r][2 * d + 1][4 * e + k] = odd;
                                }
                            }
                    } else {
                        const uint16_t* vr = reinterpret_cast<const uint16_t*>(row) + 128 * vw + 4 * half;
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float x = T::up(vr[32 * d + 8 * (e >> 2) + (e & 3)]);
                                if (seen && !(fabsf(x) < INFINITY)) acc[r][d][e] = NAN;
                            }
                    }
                }
            }
        }

        // ---- results: the two score waves of a row tile have summed half of its keys each
        lds_barrier();  // the last maxima are read
        lds_barrier();
        float ls[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r)
            ls[r] = *reinterpret_cast<const float*>(sm + L::MAX + (r * 32 + c) * 4) +
                    *reinterpret_cast<const float*>(sm + L::MAX + (MAX_ROWS + r * 32 + c) * 4);
        lds_barrier();  // free for the next segment
        if (whole) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int i = r0 + 32 * r + c;
                if (i >= r1) break;
                const float inv = ls[r] > 0.f ? 1.f / ls[r] : 0.f;
                const int t = i / a.H, h = i - t * a.H;
                uint16_t* o = static_cast<uint16_t*>(a.out) + t * a.out_row + h * a.out_head + DIMS * vw + 4 * half;
                if constexpr (Q4) {
#pragma unroll
                    for (int b = 0; b < DV / 2; ++b)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            u32x4 x;
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[j] = ls[r] == 0.f ? 0u : T::pack(acc[r][2 * b][e + j] * inv, acc[r][2 * b + 1][e + j] * inv);
                            *reinterpret_cast<u32x4*>(o + 4 * half + 64 * b + 4 * e) = x;
                        }
                } else
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<u32x2*>(o + 32 * d + 2 * e) =
                            ls[r] == 0.f ? u32x2{0u, 0u}
                                         : u32x2{T::pack(acc[r][d][e] * inv, acc[r][d][e + 1] * inv),
                                                 T::pack(acc[r][d][e + 2] * inv, acc[r][d][e + 3] * inv)};
                if (a.lse && vw == 0 && half == 0)
                    a.lse[i] = ls[r] == 0.f ? -INFINITY : (mo[r] + __builtin_amdgcn_logf(ls[r])) * 0.69314718055995f;
            }
        } else {
            // the part's slot; piece + n names a sequence's parts uniquely, since both only grow along the tiles
            const int64_t slot_bytes = (int64_t)(gr.rows / 32) * SLOT_TILE;
            const int64_t slot = prefix ? (int64_t)id : ((int64_t)piece + n) * gr.groups + g;
            char* out = static_cast<char*>(a.workspace) + SLOTS + (prefix ? 0 : p.pre_slots * (p.pre.rows / 32) * SLOT_TILE) + slot * slot_bytes;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if (r0 + 32 * r + c >= r1) break;
                int my = lane;  // (addresses found here: kept from before the loops they would be spilled, and their reload waits for all stores)
                asm volatile("" : "+v"(my));
                const int c = my & 31, half = my >> 5;
                char* o = out + r * SLOT_TILE + vw * 16384 + my * 16;
                if constexpr (Q4) {  // as the other form leaves them: a lane's 8 values in a row are two lanes' four
#pragma unroll
                    for (int b = 0; b < DV / 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            f32x16 &x = acc[r][2 * b], &y = acc[r][2 * b + 1];
                            char* to = out + r * SLOT_TILE + vw * (DIMS * 128) + c * 16 + ((2 * b + (e >> 1)) * 4 + 2 * (e & 1) + half) * 1024;
                            *reinterpret_cast<f32x4*>(to) = f32x4{x[4 * e], y[4 * e], x[4 * e + 1], y[4 * e + 1]};
                            *reinterpret_cast<f32x4*>(to + 512) = f32x4{x[4 * e + 2], y[4 * e + 2], x[4 * e + 3], y[4 * e + 3]};
                        }
                } else
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<f32x4*>(o + (d * 4 + e) * 1024) =
                            f32x4{acc[r][d][4 * e], acc[r][d][4 * e + 1], acc[r][d][4 * e + 2], acc[r][d][4 * e + 3]};
                if (vw == 0 && half == 0) *reinterpret_cast<f32x2*>(out + r * SLOT_TILE + SLOT_ACC + c * 8) = f32x2{mo[r], ls[r]};
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ joining the parts
// For 32 rows and 32 values of a sequence, two parts at a time.  SPLIT: a workgroup of 16 waves, wave v takes the parts v, v + 16,
// ..., and their sums meet in LDS (few rows with many parts: one sequence in 44 parts 5.4 us, in 4 waves 7.4; 4.5 where the
// cut is read and not found again).  Otherwise every one
// of 4 waves has a block of 32 values of its own and all parts (4096 rows: 11.2 us; with four waves to a block as above 12.4, much of it
// for finding out what there is to do).
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 1024 : 256) join_kernel(KdaLatentDecodeArgs a, Plan p) {
    constexpr int W = SPLIT ? 16 : 1;  // waves to a block
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), v = SPLIT ? w : 0, lane = tid & 63;
    const int c = lane & 31, half = lane >> 5;
    const int n = __builtin_amdgcn_readfirstlane(blockIdx.x / p.own.groups), g = blockIdx.x - n * p.own.groups;
    asm volatile("" ::"s"(a.q_latent), "s"(a.ql_row), "s"(a.page_stride), "s"(a.B), "s"(p.grid));  // all arguments at once
    const int rt = blockIdx.y / (SPLIT ? 16 : 4), block = SPLIT ? blockIdx.y & 15 : (blockIdx.y & 3) * 4 + w;  // values 32 block ..
    const Lengths lens(a);
    const u32x2 cu = *static_cast<const u32x2*>(a.workspace);
    uint32_t before = 0;
    for (int i = lane; i < n; i += 64) before += units_of(lens.of_lane(i));
    before = sum_wave(before);
    const uint32_t tiles = tiles_of(lens.of(n)), run = __builtin_amdgcn_readfirstlane(cu.x);
    const uint32_t p0 = (before + LEAD) / run, p1 = tiles ? (before + LEAD + tiles - 1) / run + 1 : p0;
    const uint32_t parts = p1 - p0, pre_parts = __builtin_amdgcn_readfirstlane(cu.y);
    if (pre_parts == 0 && parts == 1) return;  // written by the workgroup that had it whole
    const int rows = a.S * a.H;
    const int rq = g * p.own.rows + 32 * rt;  // within the sequence
    if (rq >= rows) return;
    const int r = n * rows + rq + c;
    const bool valid = rq + c < rows && 32 * rt < p.own.rows;

    float m = M_START, l = 0.f;
    f32x4 acc[4] = {};
    struct Part {
        f32x2 ml;
        f32x4 x[4];
    };
    auto load = [&](const char* slot_tile, int cc) {
        Part y;
        y.ml = *reinterpret_cast<const f32x2*>(slot_tile + SLOT_ACC + cc * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y.x[e] = *reinterpret_cast<const f32x4*>(slot_tile + (block * 4 + e) * 1024 + (32 * half + cc) * 16);
        return y;
    };
    auto add = [&](const Part& y) {
        const float mn = fmaxf(m, y.ml.x);
        const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(y.ml.x - mn);
        m = mn;
        l = l * f0 + y.ml.y * f1;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = acc[e] * f0 + y.x[e] * f1;
    };
    auto walk = [&](const char* at, int64_t step, uint32_t n, int cc) {
        uint32_t i = v;
        for (; i + W < n; i += 2 * W) {
            const Part y0 = load(at + i * step, cc), y1 = load(at + (i + W) * step, cc);
            add(y0);
            add(y1);
        }
        for (; i < n; i += W) add(load(at + i * step, cc));
    };
    if (valid) {
        const char* ws = static_cast<const char*>(a.workspace) + SLOTS;
        const int64_t own_bytes = (int64_t)(p.own.rows / 32) * SLOT_TILE, pre_bytes = (int64_t)(p.pre.rows / 32) * SLOT_TILE;
        walk(ws + p.pre_slots * pre_bytes + rt * SLOT_TILE + (((int64_t)p0 + n) * p.own.groups + g) * own_bytes, p.own.groups * own_bytes,
             parts, c);
        if (pre_parts) {
            const int gp = r / p.pre.rows, rp = r - gp * p.pre.rows;
            walk(ws + gp * pre_bytes + (rp >> 5) * SLOT_TILE, p.pre.groups * pre_bytes, pre_parts, rp & 31);
        }
    }
    auto write = [&](int at, f32x4 o, float M, float L) {  // values 32 block + at ..
        const float inv = L > 0.f ? 1.f / L : 0.f;
        const int t = r / a.H, h = r - t * a.H;
        uint16_t* out = static_cast<uint16_t*>(a.out) + t * a.out_row + h * a.out_head + 32 * block + at;
        *reinterpret_cast<u32x2*>(out) = L == 0.f ? u32x2{0u, 0u} : u32x2{T::pack(o[0] * inv, o[1] * inv), T::pack(o[2] * inv, o[3] * inv)};
        if (a.lse && block == 0 && at == 0) a.lse[r] = L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.69314718055995f;
    };
    if constexpr (SPLIT) {
        __shared__ float sm_m[W][32], sm_l[W][32];
        __shared__ f32x4 sm_a[W][4][64];
        if (half == 0) {
            sm_m[v][c] = m;
            sm_l[v][c] = l;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sm_a[v][e][lane] = acc[e];
        __syncthreads();
        if (!valid || v >= 4) return;
        float M = M_START, L = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) M = fmaxf(M, sm_m[i][c]);
        f32x4 o = {};
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float f = __builtin_amdgcn_exp2f(sm_m[i][c] - M);
            L += sm_l[i][c] * f;
            o += sm_a[i][v][lane] * f;
        }
        write(8 * v + 4 * half, o, M, L);  // wave v finishes values 8 v .. 8 v + 7 of the block
    } else if (valid) {
#pragma unroll
        for (int e = 0; e < 4; ++e) write(8 * e + 4 * half, acc[e], m, l);
    }
}

int check_decode_sizes(const KdaLatentDecodeArgs* a) {
    KDA_CHECK_ARG(a != nullptr, "latent_decode: null args");
    KDA_CHECK_ARG(a->B >= 0 && a->S >= 1 && a->H >= 1 && a->page_size >= 1 && a->table_width >= 0 && a->prefix_width >= 0 &&
                      a->num_cus >= 0 && a->num_cus <= 65536,
                  "latent_decode: B=%d S=%d H=%d page_size=%d table_width=%d prefix_width=%d num_cus=%d", a->B, a->S, a->H,
                  a->page_size, a->table_width, a->prefix_width, a->num_cus);
    KDA_CHECK_ARG((int64_t)a->S * a->H < (1ll << 31) && (int64_t)a->B * a->S * a->H < (1ll << 29) && a->B < (1 << 22),
                  "latent_decode: B * S * H is too large");
    const int64_t span = (int64_t)a->table_width * a->page_size;
    KDA_CHECK_ARG(span < (1ll << 31) && (int64_t)a->prefix_width * a->page_size < (1ll << 31),
                  "latent_decode: a table spans 2^31 tokens or more");
    KDA_CHECK_ARG(a->table_width < (1 << 28) && a->prefix_width < (1 << 28), "latent_decode: a table of 2^28 pages or more");
    KDA_CHECK_ARG(a->B * (span / BN + 1 + LEAD) < (1ll << 31), "latent_decode: the tables span 2^36 tokens or more");
    return 0;
}

Plan plan_of(const KdaLatentDecodeArgs* a) {
    Plan p;
    const int cus = a->num_cus ? a->num_cus : 256;
    // Groups of 64 rows read the keys least often.  Of 32 rows, and with a kernel for one row tile, whose steps take about two thirds
    // of the time, where even tables full of tokens leave workgroups over: 8 sequences of 12 heads behind 2000 shared tokens 15.2 us
    // instead of 17.1.
    const int64_t rows = (int64_t)a->S * a->H, own = a->B * (((int64_t)a->table_width * a->page_size + BN - 1) / BN + LEAD);
    const int64_t pre = ((int64_t)a->prefix_width * a->page_size + BN - 1) / BN;
    auto plan = [&](int most) {
        p.own = Groups::of(rows, most);
        p.pre = a->prefix_width ? Groups::of(a->B * rows, most) : Groups{32, 0};
        return p.own.groups * ((own + MIN_RUN - 1) / MIN_RUN) + p.pre.groups * ((pre + MIN_RUN - 1) / MIN_RUN);
    };
    if (plan(32) > cus) plan(MAX_ROWS);
    p.grid = cus > p.own.groups + p.pre.groups ? cus : p.own.groups + p.pre.groups;
    p.per_wg = 1.f / p.grid;
    p.pre_slots = p.pre.groups ? p.grid : 0;
    p.page = PageOf::by(a->page_size);
    return p;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int64_t kda355_latent_decode_workspace_bytes(const KdaLatentDecodeArgs* a) {
    if (const int rc = check_decode_sizes(a)) return rc;
    if (a->B == 0) return 0;
    const Plan p = plan_of(a);
    const int64_t own = p.grid + (int64_t)a->B * p.own.groups;
    return SLOTS + (p.pre_slots * (p.pre.rows / 32) + own * (p.own.rows / 32)) * SLOT_TILE;
}

namespace {
template <bool Q4>
int decode_launch(const KdaLatentDecodeArgs* a, kda355_stream_t stream) {
    if (const int rc = check_decode_sizes(a)) return rc;
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "latent_decode: dtype %d", a->dtype);
    KDA_CHECK_ARG(a->flags == 0, "latent_decode: unknown flags 0x%x", a->flags);
    if (a->B == 0) return 0;
    KDA_CHECK_ARG(a->q_latent && a->q_pe && a->cache && a->block_table && a->seq_lens && a->out && a->table_width >= 1,
                  "latent_decode: a required pointer is null");
    KDA_CHECK_ARG(a->prefix_table ? a->prefix_len && a->prefix_width >= 1 : a->prefix_width == 0,
                  "latent_decode: prefix_table needs prefix_len and prefix_width");
    KDA_CHECK_ARG(a->pages >= 1 && a->table_stride >= a->table_width, "latent_decode: pages=%lld table_stride=%lld",
                  (long long)a->pages, (long long)a->table_stride);
    KDA_CHECK_ARG(rows16(a->q_latent, a->ql_row, a->ql_head) && rows16(a->q_pe, a->qp_row, a->qp_head) &&
                      rows16(a->out, a->out_row, a->out_head),
                  "latent_decode: q and out rows must be 16-byte aligned");
    KDA_CHECK_ARG((Q4 ? aligned(a->cache, 16) && a->page_stride % 16 == 0 : rows16(a->cache, a->page_stride)) &&
                      a->page_stride >= (int64_t)a->page_size * (Q4 ? ROW4 : ROW),
                  "latent_decode: cache pages must be dense and 16-byte aligned");
    KDA_CHECK_ARG(a->scale > 0.f, "latent_decode: scale must be positive");
    const int64_t need = kda355_latent_decode_workspace_bytes(a);
    KDA_CHECK_ARG(a->workspace && aligned(a->workspace, 256) && a->workspace_bytes >= need,
                  "latent_decode: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const Plan p = plan_of(a);
    const uint32_t join = (uint32_t)a->B * p.own.groups, tiles = p.own.rows / 32;
    const bool few = (int64_t)join * tiles * 16 <= p.grid;  // blocks of rows and values: likely many parts each
    auto launch = [&](auto type) {
        typedef decltype(type) T;
        const bool two = p.own.rows > 32 || p.pre.rows > 32;  // (one row tile: one sequence of 4097 tokens, 12 heads 14.0 us, with two 15.4)
        const dim3 threads(two ? THREADS<2, Q4> : THREADS<1, Q4>);
        if (Q4 && a->page_size % 8 == 0)
            launch_kernel(two ? decode_kernel<T, 2, Q4, Q4> : decode_kernel<T, 1, Q4, Q4>, dim3(p.grid), threads, s, *a, p);
        else
            launch_kernel(two ? decode_kernel<T, 2, Q4, false> : decode_kernel<T, 1, Q4, false>, dim3(p.grid), threads, s, *a, p);
        if (few)
            launch_kernel((join_kernel<T, true>), dim3(join, tiles * 16), dim3(1024), s, *a, p);
        else
            launch_kernel((join_kernel<T, false>), dim3(join, tiles * 4), dim3(256), s, *a, p);
    };
    if (a->dtype == KDA355_DTYPE_BF16) launch(Bf16{}); else launch(Fp16{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("latent_decode: launch failed: %s", hipGetErrorString(e));
        return KDA355_ELAUNCH;
    }
    return 0;
}
}  // namespace

extern "C" int kda355_latent_decode_launch(const KdaLatentDecodeArgs* a, kda355_stream_t stream) { return decode_launch<false>(a, stream); }
extern "C" int kda355_latent4_decode_launch(const KdaLatentDecodeArgs* a, kda355_stream_t stream) { return decode_launch<true>(a, stream); }
