// Latent attention, expanded form (gfx950): per-head keys of 128 | 64 (the 64 shared by the heads) and values of 128 over
// packed sequences, causal or not.
//
// A workgroup of 4 wave64 takes 128 query rows of one (sequence, head), 32 a wave, and walks the keys in tiles of 64:
// keys, shared parts and values come straight into LDS (40 KiB a tile, two tiles, so two workgroups share a CU), one barrier
// a tile, the next tile's loads under way while this one is computed.  Per wave and tile: scores 24 MFMAs, running softmax
// in registers, values 16 MFMAs (attend.h has the layouts).
//
// Bound: the matrix cores (40 MFMAs of 32 cycles a wave and tile, two waves a SIMD), and while they run the card's power: the clock
// stands at 1.75 GHz where a kernel bound by HBM keeps 2.3 to 2.4.  8192 causal tokens of 32 heads: 639 to 686 us on different cards,
// 1.00 to 1.08 of the 1.22 PFLOP/s that a large library product reaches (754 in the first 20 passes after a pause); the matrix cores are
// busy 62 % of the cycles, LDS reads (4 cycles for 1 KiB, no conflicts) 31 %, and with fewer waits the clock falls as much as the cycles
// (operands read 8 steps ahead: 10 % fewer cycles, the same time).  64 rows a wave, one wave a SIMD: 680 us against 651 then, a wave
// issues an instruction every 5.6 cycles at best.  Six prompts of 1 to 2048 tokens with up to 8191 before them: 161 us (207 soon
// after a pause), a tile of 128 rows as fast as above, but a quarter of the tiles has few rows, and their waves without any row do the
// matrix steps of the others (17 % of all here); the last 25 us have few workgroups.  77 rows of 16 heads over 1277 keys: 15.4 us,
// of which 4.5 join the pieces and 4.8 go by in a piece's three tiles, one after the other; most of the rest is the start.
#include <type_traits>

#include "attend.h"

namespace kda355 {
namespace {

constexpr int BM = 128, BN = 64, WAVES = 4;
constexpr int HD = 128, PE = 64;
constexpr int TILE_V = BN * HD * 2, TILE_PE = 2 * TILE_V, TILE_BYTES = TILE_PE + BN * PE * 2;  // k | v | shared part
constexpr int SLOT_ACC = BM * HD * 4, SLOT = SLOT_ACC + BM * 8;  // workspace of a part: accumulators, (m, l) of each row
// Where rows are few and keys many, the keys are cut: a sequence whose last row tile sees more key tiles than a workgroup's fair
// share of all (and than MIN_RUN) has every row tile walked in that many pieces, whose parts a second kernel joins.  (77 rows over
// 1277 keys, 16 heads: 16.0 us in pieces of 2 tiles, 15.3 of 3, 17.3 of 4.)
constexpr int MIN_RUN = 3;
constexpr int64_t MAX_ROW = 1 << 23;  // row strides up to this many elements: a tile's byte offsets stay below 2^31

struct Plan { int grid, share, slots; };  // workgroups; those that share the work; parts in the workspace
struct Seq {
    int tiles, most, pieces;  // row tiles; key tiles of the last one; pieces of each
};
struct Span {
    int q0, k0;         // (below 2^30)
    int Lq, Lk, shift;  // row i sees keys j <= i + shift, j < Lk
};
__device__ __forceinline__ Span span_of(const KdaLatentPrefillArgs& a, int n) {
    const int Tq = (int)a.Tq, Tk = (int)a.Tk;
    Span s;
    s.q0 = min(max(a.cu_q[n], 0), Tq), s.k0 = min(max(a.cu_k[n], 0), Tk);
    s.Lq = max(min(a.cu_q[n + 1], Tq) - s.q0, 0), s.Lk = max(min(a.cu_k[n + 1], Tk) - s.k0, 0);
    s.shift = a.flags & KDA355_LATENT_CAUSAL ? s.Lk - s.Lq : s.Lk;
    return s;
}
// key tiles that row tile `i` sees
__device__ __forceinline__ int key_tiles(const Span& s, int i) {
    const int seen = min(s.Lk, min(i * BM + BM, s.Lq) + s.shift);
    return seen > 0 ? (seen + BN - 1) / BN : 0;
}
// key tiles of a piece of a row tile that sees `n` of them
__device__ __forceinline__ int run_of(int n, int pieces) { return max((n + pieces - 1) / pieces, MIN_RUN); }
// every lane takes a sequence; the first 64 are loaded once
struct Spans {
    const KdaLatentPrefillArgs& a;
    Span mine;
    __device__ __forceinline__ explicit Spans(const KdaLatentPrefillArgs& args) : a(args), mine(span_of(args, min((int)(threadIdx.x & 63), args.N - 1))) {}
    __device__ __forceinline__ Span operator[](int n) const { return n < 64 ? mine : span_of(a, n); }  // n % 64: the lane
    __device__ __forceinline__ Span of(int n) const {                                                  // n: the same in all lanes
        const Span s = n < 64 ? mine : span_of(a, n);
        const int l = n < 64 ? n : 0;
        return {__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.k0, l), __builtin_amdgcn_readlane(s.Lq, l),
                __builtin_amdgcn_readlane(s.Lk, l), __builtin_amdgcn_readlane(s.shift, l)};
    }
};
// The longest run of a piece: a fair share of the key tiles of all row tiles (about).
__device__ __forceinline__ int longest_run(const KdaLatentPrefillArgs& a, const Spans& spans, int slots) {
    const int lane = threadIdx.x & 63;
    float all = 0.f;
    for (int n = lane; n < a.N; n += 64) {
        const Span s = spans[n];
        const int tiles = (s.Lq + BM - 1) / BM;
        if (tiles) all += (float)tiles * (0.5f * (key_tiles(s, 0) + key_tiles(s, tiles - 1)));
    }
    return __builtin_amdgcn_readfirstlane(max((int)fminf(__builtin_ceilf(sum_wave(all) * a.H / slots), 1e9f), MIN_RUN));
}
__device__ __forceinline__ Seq seq_of(const Span& s, int run) {
    Seq q;
    q.tiles = (s.Lq + BM - 1) / BM;
    q.most = q.tiles ? key_tiles(s, q.tiles - 1) : 0;
    q.pieces = max((q.most + run - 1) / run, 1);
    return q;
}
// The pieces of 64 sequences, one a lane, with what the lanes before it and itself have together.
struct Pieces {
    Seq q;
    int pieces, parts, split;
};
__device__ __forceinline__ Pieces pieces_of(const KdaLatentPrefillArgs& a, const Spans& spans, int run, int n) {
    Pieces p;
    p.q = n < a.N ? seq_of(spans[n], run) : Seq{0, 0, 1};
    const bool cut = p.q.pieces > 1;
    p.pieces = scan_wave(p.q.tiles * p.q.pieces);
    p.parts = scan_wave(cut ? p.q.tiles * p.q.pieces : 0);
    p.split = scan_wave(cut ? p.q.tiles : 0);
    return p;
}
// What all workgroups find alike: the longest run, and of a head all pieces, the pieces of split row tiles, and those row tiles.
struct Cut {
    int run, pieces, parts, split;
    Pieces first;  // the first 64 sequences
};
__device__ __forceinline__ Cut cut(const KdaLatentPrefillArgs& a, const Spans& spans, const Plan& p) {
    const int lane = threadIdx.x & 63;
    Cut c;
    c.run = longest_run(a, spans, p.share);
    for (int again = 0; again < 2; ++again) {
        c.pieces = c.parts = c.split = 0;
        for (int n0 = 0; n0 < a.N; n0 += 64) {
            const Pieces x = pieces_of(a, spans, c.run, n0 + lane);
            if (n0 == 0) c.first = x;
            c.pieces += __builtin_amdgcn_readlane(x.pieces, 63);
            c.parts += __builtin_amdgcn_readlane(x.parts, 63);
            c.split += __builtin_amdgcn_readlane(x.split, 63);
        }
        // (always so, but for the rounding of the sum: pieces <= row tiles + 2 share / H, parts <= 4 share / H)
        if ((int64_t)c.pieces * a.H <= p.grid && (int64_t)c.parts * a.H <= p.slots) break;
        c.run = 1 << 30;
    }
    return c;
}
struct Where {
    int n, tile, piece, pieces;  // sequence, row tile, piece of it, pieces of the row tile
    int slot;                    // of the row tile's first piece among the split ones of the head
};
// Piece `i` of a head (SPLIT: split row tile i); n < 0 past the last one.
template <bool SPLIT>
__device__ __forceinline__ Where locate(const KdaLatentPrefillArgs& a, const Spans& spans, const Cut& c, int i) {
    const int lane = threadIdx.x & 63;
    int before = 0, parts_before = 0;
    for (int n0 = 0; n0 < a.N; n0 += 64) {
        const Pieces x = n0 == 0 ? c.first : pieces_of(a, spans, c.run, n0 + lane);
        const int s = SPLIT ? x.split : x.pieces, all = x.q.tiles * x.q.pieces;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(before + s > i);
        if (hit) {
            const int l = __builtin_ctzll(hit), pieces = __builtin_amdgcn_readlane(x.q.pieces, l);
            const int parts = pieces > 1 ? __builtin_amdgcn_readlane(all, l) : 0;
            const int mine = SPLIT ? __builtin_amdgcn_readlane(x.q.tiles, l) : __builtin_amdgcn_readlane(all, l);
            const int at = i - before - (__builtin_amdgcn_readlane(s, l) - mine);
            Where w;
            w.n = n0 + l;
            w.pieces = pieces;
            w.tile = SPLIT ? at : at / pieces;
            w.piece = SPLIT ? 0 : at - w.tile * pieces;
            w.slot = parts_before + __builtin_amdgcn_readlane(x.parts, l) - parts + w.tile * pieces;
            return w;
        }
        before += __builtin_amdgcn_readlane(s, 63);
        parts_before += __builtin_amdgcn_readlane(x.parts, 63);
    }
    return {-1, 0, 0, 1, 0};
}

template <typename T>
__global__ void __launch_bounds__(WAVES * 64, 2) prefill_kernel(KdaLatentPrefillArgs a, Plan p) {
    __shared__ __align__(1024) unsigned char sm[2 * TILE_BYTES];
    asm volatile("" ::"s"(a.q), "s"(a.q_row), "s"(a.Tq), "s"(a.num_cus), "s"(p.grid));  // all arguments at once
    const Spans spans(a);
    const Cut cu = cut(a, spans, p);
    if ((int64_t)blockIdx.x >= (int64_t)cu.pieces * a.H) return;
    // A piece of all heads side by side, long walks first (the last of a causal sequence), so that what starts last is short.
    // With 8 heads or a multiple, a head stays on one XCD, whose L2 its keys pass.  (A head's pieces side by side and few heads
    // at a time: 8192 causal tokens, 32 heads 700 us instead of 659.)
    const int i = __builtin_amdgcn_readfirstlane(blockIdx.x / a.H), h = __builtin_amdgcn_readfirstlane(blockIdx.x - i * a.H);
    const Where at = locate<false>(a, spans, cu, cu.pieces - 1 - i);
    const int n = __builtin_amdgcn_readfirstlane(at.n);
    if (n < 0) return;
    const int m0 = __builtin_amdgcn_readfirstlane(at.tile) * BM;
    const Span sp = spans.of(n);
    const int64_t q0 = sp.q0, k0 = sp.k0;
    const int Lq = sp.Lq, Lk = sp.Lk, shift = sp.shift;
    const int ntiles = __builtin_amdgcn_readfirstlane(key_tiles(sp, at.tile));
    const int length = run_of(ntiles, at.pieces), first = __builtin_amdgcn_readfirstlane(at.piece * length);
    const int last = __builtin_amdgcn_readfirstlane(min(first + length, ntiles));  // this piece's key tiles
    if (at.piece > 0 && first >= ntiles) return;  // (a short row tile of a split sequence; the join counts its pieces alike)
    const bool part = ntiles > length;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 31, half = lane >> 5;
    const int row = m0 + 32 * w + c;

    // ---- tile loads: wave w brings tokens 16 w .. 16 w + 15
    const uint16_t* kh = static_cast<const uint16_t*>(a.k) + k0 * a.k_row + h * a.k_head;
    const uint16_t* vh = static_cast<const uint16_t*>(a.v) + k0 * a.v_row + h * a.v_head;
    const uint16_t* ph = static_cast<const uint16_t*>(a.k_pe) + k0 * a.pe_row;
    const uint32_t lds = lds_offset(sm);
    uint32_t koff[4], voff[4], poff[2];  // byte offsets of this lane's pieces (k / v load i: tokens 16 w + 4 i ..; swz16)
    const int lt = 16 * w + (lane >> 4), pt = 16 * w + (lane >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t piece = ((lane & 15) ^ ((lane >> 4) << 2) ^ i) * 16;
        koff[i] = (uint32_t)(lt + 4 * i) * (uint32_t)(2 * a.k_row) + piece;
        voff[i] = (uint32_t)(lt + 4 * i) * (uint32_t)(2 * a.v_row) + piece;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) poff[i] = (uint32_t)(pt + 8 * i) * (uint32_t)(2 * a.pe_row) + ((lane & 7) ^ swz8(pt + 8 * i)) * 16;
    // A tile's descriptors end with the row of its last token, so that tokens past it read as zeros (where rows overlap or are
    // one and the same: as its values, and like the zeros they are hidden).
    struct Tile { u32x4 k, v, pe; uint32_t at; };
    const uint32_t krow = 2 * (uint32_t)a.k_row, vrow = 2 * (uint32_t)a.v_row, prow = 2 * (uint32_t)a.pe_row;
    const char* kn = reinterpret_cast<const char*>(kh) + (int64_t)first * BN * krow;  // the next tile to be brought
    const char* vn = reinterpret_cast<const char*>(vh) + (int64_t)first * BN * vrow;
    const char* pn = reinterpret_cast<const char*>(ph) + (int64_t)first * BN * prow;
    auto tile_at = [&](int j) {  // called for one after the other
        const bool whole = j * BN + BN <= Lk, some = j < last;  // past the piece: nothing is read
        const uint32_t n = whole ? BN - 1 : Lk - j * BN - 1;
        Tile t;
        t.k = tile_rsrc(kn, some ? n * krow + HD * 2 : 0);
        t.v = tile_rsrc(vn, some ? n * vrow + HD * 2 : 0);
        t.pe = tile_rsrc(pn, some ? n * prow + PE * 2 : 0);
        t.at = lds + (j & 1) * TILE_BYTES + 16 * w * (HD * 2);
        kn += BN * (int64_t)krow, vn += BN * (int64_t)vrow, pn += BN * (int64_t)prow;
        return t;
    };
    auto bring = [&](const Tile& t, int i) {  // load i of 10
        if (i < 4)
            load_to_lds(t.at + 4 * i * (HD * 2), t.k, koff[i]);
        else if (i < 8)
            load_to_lds(t.at + TILE_V + 4 * (i - 4) * (HD * 2), t.v, voff[i - 4]);
        else
            load_to_lds(t.at - 16 * w * (HD * 2) + TILE_PE + (16 * w + 8 * (i - 8)) * (PE * 2), t.pe, poff[i - 8]);
    };

    // ---- LDS read addresses (byte offsets within a tile; key step, value tile and key block are xors and constants)
    const uint32_t ka = c * (HD * 2) + ((half ^ swz16(c)) << 4);
    const uint32_t pa = TILE_PE + c * (PE * 2) + ((half ^ swz8(c)) << 4);
    const int i16 = lane & 15;
    uint32_t va[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t = 4 * half + 8 * u + (i16 >> 2);
        const int e = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
        va[u] = TILE_V + t * (HD * 2) + ((e ^ swz16(t)) << 4) + (i16 & 1) * 8;
    }

    const float sc = a.scale * 1.44269504088896f;
    f32x16 acc[4] = {};
    float mo = M_START, l = 0.f;
    bool special = false;
    const int mine = m0 + 32 * w < Lq ? min(Lk, min(m0 + 32 * w + 32, Lq) + shift) : 0;  // keys that any row of this wave sees
    const int full = min(Lk, m0 + 32 * w + 1 + shift);         // keys that every row of this wave sees
    if (first < last) {
        const Tile t = tile_at(first);
#pragma unroll
        for (int i = 0; i < 10; ++i) bring(t, i);
    }
    // ---- queries: a wave's 32 rows (past the end the last one again).  Their first 128 come through the LDS of the second tile,
    // 256 bytes a row, laid out like keys, the last 64 straight, 32 bytes of every row at a time (all of them so: 15.6 us instead of 15.3
    // for 77 rows and 1277 keys).
    u32x4 q[12] = {};
    if (m0 + 32 * w < Lq) {
        const uint16_t* qh = static_cast<const uint16_t*>(a.q) + q0 * a.q_row + h * a.q_head;
        const uint32_t at = lds + ((first + 1) & 1) * TILE_BYTES + 32 * w * (HD * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 4);
            load_block<0>(at + i * 1024, (uint64_t)(qh + min(m0 + 32 * w + r, Lq - 1) * a.q_row) + (((lane & 15) ^ swz16(r)) << 4));
        }
        const uint16_t* qr = qh + min(row, Lq - 1) * a.q_row + 8 * half;
#pragma unroll
        for (int i = 8; i < 12; ++i) q[i] = *reinterpret_cast<const u32x4*>(qr + 16 * i);
        wait_loads<0>();
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = lds_read16((at + ka) ^ (i << 5));
    }
    // the queries are there before the loop: the compiler would wait for them, and so for the next tile, in it
#pragma unroll
    for (int i = 0; i < 12; ++i) asm volatile("" : "+v"(q[i]));
    auto tile = [&](int j, auto masked_) {  // MASKED: some row of the wave does not see some key of the tile
        constexpr bool MASKED = decltype(masked_)::value;
        wait_loads<0>();
        lds_barrier();  // tile j is whole, and every wave has read tile j - 1
        const int t0 = j * BN;
        const Tile next = tile_at(j + 1);
        const uint32_t tb = lds + (j & 1) * TILE_BYTES;
        // ---- scores: 24 steps (key step i of 12, key block b of 2), the operands of the next four read while four run, the next
        // tile's loads between them
        f32x16 s[2] = {};
        auto key = [&](int x) {
            const int i = x >> 1, b = x & 1;
            return i < 8 ? lds_read16((tb + ka + b * 32 * HD * 2) ^ (i << 5)) : lds_read16((tb + pa + b * 32 * PE * 2) ^ ((i - 8) << 5));
        };
        u32x4 kf[2][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) kf[0][x] = key(x);
#pragma unroll
        for (int g = 0; g < 6; ++g) {
            __builtin_amdgcn_sched_barrier(0);
            if (g < 5)
#pragma unroll
                for (int x = 0; x < 4; ++x) kf[(g + 1) & 1][x] = key(4 * g + 4 + x);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[x & 1] = T::mfma(kf[g & 1][x], q[2 * g + (x >> 1)], s[x & 1]);
                if (g < 5 && (x & 1)) bring(next, 2 * g + (x >> 1));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MASKED) {
            const int seen = min(row + shift, Lk - 1) - t0 - 4 * half;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * b + (r & 3) + 8 * (r >> 2) > seen) s[b][r] = -INFINITY;
        }
        // ---- running softmax: the maximum is raised, and the accumulator rescaled, only when some row of the wave
        // exceeds it by SLACK (the result is the same for any reference; weights stay within the type's range)
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        mx = max_halves(mx) * sc;
        if (__builtin_amdgcn_ballot_w64(mx - mo > T::B + T::SLACK)) {
            const float mn = mx - mo > T::B + T::SLACK ? mx - T::B : mo;  // by the row's own scores alone
            const float f = __builtin_amdgcn_exp2f(mo - mn);
            mo = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= f;
        }
        u32x4 p[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[b][r], sc, -mo)), y = __builtin_amdgcn_exp2f(fmaf(s[b][r + 1], sc, -mo));
                l += x + y;
                p[2 * b + (r >> 3)][(r >> 1) & 3] = T::pack(x, y);
            }
        // ---- values
        auto value = [&](int k, int d) {
            const u32x2 v0 = lds_read_tr(((tb + va[0]) ^ (d << 6)) + k * 16 * HD * 2);
            const u32x2 v1 = lds_read_tr(((tb + va[1]) ^ (d << 6)) + k * 16 * HD * 2);
            return u32x4{v0.x, v0.y, v1.x, v1.y};
        };
        u32x4 vf[2][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) vf[0][d] = value(0, d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            if (k < 3)
#pragma unroll
                for (int d = 0; d < 4; ++d) vf[(k + 1) & 1][d] = value(k + 1, d);
            if constexpr (MASKED)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    special |= nonfinite<T>(vf[k & 1][d]);
                    vf[k & 1][d] = finite_part<T>(vf[k & 1][d]);
                }
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] = T::mfma(vf[k & 1][d], p[k], acc[d]);
        }
    };
    const int clean = min(last, max(full, 0) / BN), mixed = min(last, (mine + BN - 1) / BN);
    int j = first;
    for (; j < clean; ++j) tile(j, std::false_type{});
    for (; j < mixed; ++j) tile(j, std::true_type{});
    for (; j < last; ++j) {  // tiles that only later rows see
        wait_loads<0>();
        lds_barrier();
        const Tile next = tile_at(j + 1);
#pragma unroll
        for (int i = 0; i < 10; ++i) bring(next, i);
    }
    wait_loads<0>();  // (nothing is left in flight towards LDS)
    // Infinite or NaN values in tiles that not every row sees whole.  A positive weight leaves such a value as it is, however small: it is
    // added even where the weight has become 0 in fp32 (a tile that every row sees gives 0 inf = NaN there).
    if (__builtin_amdgcn_ballot_w64(special)) {
        const int seen = min(row + shift, Lk - 1);
#pragma unroll 1
        for (int j = max(max(full, 0) & ~(BN - 1), first * BN); j < min(mine, last * BN); ++j) {
            const uint16_t* vr = vh + (int64_t)j * a.v_row + 4 * half;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = T::up(vr[32 * d + 8 * g + e]);
                        if (j <= seen && !(fabsf(x) < INFINITY)) acc[d][4 * g + e] += x;
                    }
        }
    }

    l = sum_halves(l);
    if (row >= Lq) return;
    if (part) {
        char* slot = static_cast<char*>(a.workspace) + ((int64_t)h * cu.parts + at.slot + at.piece) * SLOT;
        if (half == 0) *reinterpret_cast<f32x2*>(slot + SLOT_ACC + (32 * w + c) * 8) = f32x2{mo, l};
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(slot + ((w * 4 + d) * 4 + g) * 1024 + lane * 16) =
                    f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
        return;
    }
    // ---- o = acc / l
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* o = static_cast<uint16_t*>(a.out) + (q0 + row) * a.out_row + h * a.out_head + 4 * half;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float x0 = acc[d][4 * g] * inv, x1 = acc[d][4 * g + 1] * inv, x2 = acc[d][4 * g + 2] * inv, x3 = acc[d][4 * g + 3] * inv;
            *reinterpret_cast<u32x2*>(o + 32 * d + 8 * g) =
                l == 0.f ? u32x2{0u, 0u} : u32x2{T::pack(x0, x1), T::pack(x2, x3)};
        }
    if (a.lse && half == 0)
        a.lse[(q0 + row) * a.H + h] = l == 0.f ? -INFINITY : (mo + __builtin_amdgcn_logf(l)) * 0.69314718055995f;
}

// ------------------------------------------------------------------------------------------------ joining the parts
// One workgroup for 32 rows (blockIdx.y) of a split row tile; wave d takes values 32 d .., parts two at a time.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(KdaLatentPrefillArgs a, Plan p) {
    const Spans spans(a);
    const Cut cu = cut(a, spans, p);
    for (int64_t task = blockIdx.x; task < (int64_t)cu.split * a.H; task += gridDim.x) {
        const int h = __builtin_amdgcn_readfirstlane((int)(task / cu.split));
        const Where at = locate<true>(a, spans, cu, (int)(task - (int64_t)h * cu.split));
        const Span sp = spans.of(__builtin_amdgcn_readfirstlane(at.n));
        const int ntiles = key_tiles(sp, at.tile), length = run_of(ntiles, at.pieces);
        if (ntiles <= length) continue;  // one piece: written by its workgroup
        const int parts = __builtin_amdgcn_readfirstlane((ntiles + length - 1) / length);
        const int d = threadIdx.x >> 6, lane = threadIdx.x & 63, w = blockIdx.y, c = lane & 31, half = lane >> 5;
        const int row = at.tile * BM + 32 * w + c;
        if (row >= sp.Lq) continue;
        const char* slot = static_cast<const char*>(a.workspace) + ((int64_t)h * cu.parts + at.slot) * SLOT;
        struct Part {
            f32x2 ml;
            f32x4 x[4];
        };
        auto load = [&](int i) {
            Part y;
            y.ml = *reinterpret_cast<const f32x2*>(slot + (int64_t)i * SLOT + SLOT_ACC + (32 * w + c) * 8);
#pragma unroll
            for (int g = 0; g < 4; ++g) y.x[g] = *reinterpret_cast<const f32x4*>(slot + (int64_t)i * SLOT + ((w * 4 + d) * 4 + g) * 1024 + lane * 16);
            return y;
        };
        float m = M_START, l = 0.f;
        f32x4 acc[4] = {};
        auto add = [&](const Part& y) {
            const float mn = fmaxf(m, y.ml.x);
            const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(y.ml.x - mn);
            m = mn;
            l = l * f0 + y.ml.y * f1;
#pragma unroll
            for (int g = 0; g < 4; ++g) acc[g] = acc[g] * f0 + y.x[g] * f1;
        };
        int i = 0;
        for (; i + 1 < parts; i += 2) {
            const Part y0 = load(i), y1 = load(i + 1);
            add(y0);
            add(y1);
        }
        if (i < parts) add(load(i));
        const float inv = l > 0.f ? 1.f / l : 0.f;
        uint16_t* o = static_cast<uint16_t*>(a.out) + ((int64_t)sp.q0 + row) * a.out_row + h * a.out_head + 32 * d + 4 * half;
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x2*>(o + 8 * g) =
                l == 0.f ? u32x2{0u, 0u} : u32x2{T::pack(acc[g][0] * inv, acc[g][1] * inv), T::pack(acc[g][2] * inv, acc[g][3] * inv)};
        if (a.lse && d == 0 && half == 0)
            a.lse[((int64_t)sp.q0 + row) * a.H + h] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055995f;
    }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// rows of 16-byte pieces: aligned base, strides in multiples of 8 elements
bool rows16(const void* p, int64_t s0, int64_t s1 = 0) { return aligned(p, 16) && s0 % 8 == 0 && s1 % 8 == 0; }
bool near(int64_t row) { return row >= 0 && row <= MAX_ROW; }

}  // namespace
}  // namespace kda355

using namespace kda355;

static int check_prefill_sizes(const KdaLatentPrefillArgs* a) {
    KDA_CHECK_ARG(a != nullptr, "latent_prefill: null args");
    KDA_CHECK_ARG(a->N >= 0 && a->H >= 1 && a->Tq >= 0 && a->Tk >= 0 && a->num_cus >= 0 && a->num_cus <= 65536,
                  "latent_prefill: N=%d H=%d Tq=%lld Tk=%lld num_cus=%d", a->N, a->H, (long long)a->Tq, (long long)a->Tk, a->num_cus);
    KDA_CHECK_ARG(a->Tq < (1ll << 30) && a->Tk < (1ll << 30), "latent_prefill: 2^30 tokens or more");
    KDA_CHECK_ARG((a->Tq / BM + a->N) * a->H < (1ll << 22), "latent_prefill: grid too large");
    return 0;
}
static Plan plan_of(const KdaLatentPrefillArgs* a) {
    const int64_t rows = (a->Tq / BM + a->N) * a->H;  // at least the row tiles of all sequences and heads
    Plan p;
    p.share = 2 * (a->num_cus ? a->num_cus : 256);  // two workgroups a CU
    p.grid = (int)(rows + 2 * p.share);
    const int64_t most = rows * ((a->Tk / BN + 1 + MIN_RUN - 1) / MIN_RUN);
    p.slots = (int)(most < 4 * p.share ? most : 4 * p.share);
    return p;
}

extern "C" int64_t kda355_latent_prefill_workspace_bytes(const KdaLatentPrefillArgs* a) {
    if (const int rc = check_prefill_sizes(a)) return rc;
    if (a->N == 0 || a->Tq == 0) return 0;
    return (int64_t)plan_of(a).slots * SLOT;
}

extern "C" int kda355_latent_prefill_launch(const KdaLatentPrefillArgs* a, kda355_stream_t stream) {
    if (const int rc = check_prefill_sizes(a)) return rc;
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "latent_prefill: dtype %d", a->dtype);
    KDA_CHECK_ARG((a->flags & ~KDA355_LATENT_CAUSAL) == 0, "latent_prefill: unknown flags 0x%x", a->flags);
    if (a->N == 0 || a->Tq == 0) return 0;
    KDA_CHECK_ARG(a->q && a->out && a->cu_q && a->cu_k && (a->Tk == 0 || (a->k && a->v && a->k_pe)),
                  "latent_prefill: a required pointer is null");
    KDA_CHECK_ARG(rows16(a->q, a->q_row, a->q_head) && rows16(a->k, a->k_row, a->k_head) && rows16(a->v, a->v_row, a->v_head) &&
                      rows16(a->k_pe, a->pe_row) && rows16(a->out, a->out_row, a->out_head),
                  "latent_prefill: rows must be 16-byte aligned");
    KDA_CHECK_ARG(near(a->k_row) && near(a->v_row) && near(a->pe_row), "latent_prefill: token strides of k, v and k_pe must be at most 2^23");
    KDA_CHECK_ARG(a->scale > 0.f, "latent_prefill: scale must be positive");
    const int64_t need = kda355_latent_prefill_workspace_bytes(a);
    KDA_CHECK_ARG(a->workspace && aligned(a->workspace, 256) && a->workspace_bytes >= need,
                  "latent_prefill: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const Plan p = plan_of(a);
    const dim3 join(p.slots / 2 < 1 ? 1 : min(p.slots / 2, p.share), WAVES);  // a split row tile has two parts at least
    auto launch = [&](auto type) {
        typedef decltype(type) T;
        launch_kernel(prefill_kernel<T>, dim3(p.grid), dim3(WAVES * 64), s, *a, p);
        launch_kernel(join_kernel<T>, join, dim3(256), s, *a, p);
    };
    if (a->dtype == KDA355_DTYPE_BF16) launch(Bf16{}); else launch(Fp16{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("latent_prefill: launch failed: %s", hipGetErrorString(e));
        return KDA355_ELAUNCH;
    }
    return 0;
}
