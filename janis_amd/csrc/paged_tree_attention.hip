// Attention of trees of drafted tokens over a paged key/value cache (jh_paged_tree_attention),
// on the parts that it shares with jh_paged_attention: there, what a tile does with a part of
// its keys is described. Here a new token sees the committed keys of its request and, of the
// new ones, those whose bits its mask has; the tiles that meet new keys take the bits of 32
// keys as one word per row.
//
// Trees have some dozens to hundreds of rows (new tokens times the query heads of a kv head)
// over caches of very different lengths, which is too few tiles to fill the GPU and too
// unequal to deal them out. So the work is dealt out instead: all tiles of a kv head, each
// its 64-key units times what a unit of its kind costs, stand in one line, which is cut into
// as many pieces of equal cost as blocks are resident. A block finds its piece by running sums over
// the requests and walks it: the end of one tile, whole ones, the beginning of another. A
// tile that is cut leaves parts, which a launch that follows joins in their order (joined by
// the part that arrives last, the largest tiles, of 128 rows in 30 parts, held one block for
// 170 us, and the launch is 4 to 20). A cut near a tile's end is moved there.
//
// Equal cost is not equal time: of the blocks of 63 tokens over 30000 keys, whose pieces are
// alike, the fastest took 37 us, half of them 47 and the slowest 55; of those of 64 requests 105, 156 and
// 190. And all tiles of a run (n > 32 * mask_words) are charged all of its keys, though an early
// one ends at its rows' own: 2000 tokens of 2000 87 us, jh_paged_attention 70; of 8000 327 and 313.
//
// What bounds it, bf16, 32 heads on 8 of 128 (MI355X):
//   16 tokens of 700 keys    14.5 us: round trips (lengths, the line, tables, keys, records), 11
//     of them the parts and 4 the launch that joins
//   63 of 30000              66 to 73 us, by device: 58 the parts, 8 the join; MFMA, two thirds of it
//     the second product made twice, at a clock that the power holds to 1.8 GHz
//   64 requests of 20 to 60 over 100 to 8000 208 to 220 us, by device (413 TFLOP/s of the formula's
//     operations in all, tiles that are not full not counted): 19 to 22 the join, records to memory
//     and back, the rest the parts (182 at the least, more under a profiler). The clock is 1.8 GHz of
//     2.4, by power, and the matrix pipes busy half of it
//   tiles of 32 rows alone   HBM: 64 requests of 8 tokens over 4000 keys 173 us, 6.1 TB/s
// head_dim 64 and 256: 16 requests of 32 tokens over 4000 keys 49 and 148 us (128: 78), 63 tokens over
// 30000 45 and 123 us (65).
#include "paged_attention.hpp"

namespace jh {
namespace {

// Kinds of tiles, by rows: 128 (four waves of 32 share 64 keys), 64 (two pairs of waves,
// 32 keys each), 32 (each wave takes 32 keys of its own).
struct TreeAttn {
    PagedAttnArgs a;
    int G;            // Hq / Hk
    int blocks;       // most pieces of a kv head's line
    int record, size; // rows and floats (whole 128-byte lines) of a record
    struct Split* split;  // of block b: the tile that begins there and goes on in the next; nullptr: keys stay whole
    float* part;      // records: [blocks] of the tiles that go on in a block, [blocks] of those that begin there
};
// Cost of a unit of 64 keys, by the tile's rows: with all blocks at work one takes 2.7, 3.1, 3.6 and
// 4.0 us for tiles of 32, 64, 96 and 128 rows (bf16, head_dim 128; used for f16, 64 and 256 too, where it
// was not taken apart). And of a tile (its queries, its results): 4 to 8 us.
__device__ __forceinline__ int cost_of(int rows) { return 4 + (rows + 31) / 32; }
constexpr int kCostTile = 12;
// The least cost of a piece, below which a block costs more to begin than it saves: 16 tokens over
// 700 keys (32 heads on 8) took 16.7, 19.1 and 21.1 us with 12, 24 and 36; larger calls the same.
constexpr double kLeastPiece = 12;
// The least units of a part: a cut nearer a tile's end is moved there. 16 requests of 8 to 32
// tokens over 500 to 5000 keys took 60, 58 and 63 us with 1, 2 and 4.
constexpr int kLeastUnits = 2;

// Keys up to the last one that the row sees.
__device__ __forceinline__ int reach(const PagedAttnArgs& a, const Request& q, int row, int G) {
    if (!is_tree(a, q)) return seen(q, row, G);
    const uint32_t* const m = a.mask + (int64_t)(q.start + row / G) * a.mask_words;
    int top = 0;
    for (int w = (q.n - 1) / 32; w >= 0 && top == 0; w--) {
        const uint32_t bits = q.n - 32 * w < 32 ? m[w] & ((1u << (q.n - 32 * w)) - 1) : m[w];
        if (bits) top = 32 * w + 32 - __clz((int)bits);
    }
    return max(0, q.kv - q.n + top);
}
// Of the rows up to `last`, and what all rows from `first` on see.
__device__ __forceinline__ int reach_of_tile(const PagedAttnArgs& a, const Request& q, int last, int G) {
    return is_tree(a, q) ? q.kv : seen(q, last, G);
}
__device__ __forceinline__ int seen_by_all(const PagedAttnArgs& a, const Request& q, int first, int G) {
    return is_tree(a, q) ? max(0, q.kv - q.n) : seen(q, first, G);
}

struct Split {
    int4 at;  // parts (0: no such tile), first row, rows
    int4 q;   // the request
};
struct Shape {
    int whole, rest;     // tiles of 128 rows, and rows behind them
    int rest_tiles;      // 0 or 1
    int units;
    double tile, cost;   // of a tile of 128 rows; of the request
};
__device__ __forceinline__ Shape shape_of(const Request& q, int G) {
    Shape s;
    const int rows = q.n * G;
    s.whole = rows / kManyRows, s.rest = rows % kManyRows, s.rest_tiles = s.rest > 0;
    s.units = max(1, (q.kv + kUnit - 1) / kUnit);
    s.tile = (double)s.units * cost_of(kManyRows) + kCostTile;
    s.cost = s.whole * s.tile + (s.rest ? (double)s.units * cost_of(s.rest) + kCostTile : 0.0);
    return s;
}

// A place on the line: before unit `unit` of tile `tile` of request r, which begins at `begin`.
struct Place {
    int r, tile, unit;
    double begin;
    Request q;
};
// The line's cuts: all a block keeps of it (in scalar registers).
struct Cuts {
    double each, total;  // cost of a piece, and of the line
    int pieces;
    // Where piece j (not the first behind the last) begins.
    __device__ __forceinline__ double at(int j) const { return floor(each * j); }
};
// A wave's view of the line: a lane sums a run of requests.
struct Line {
    Cuts cuts;
    double before; // the lane's run's beginning (exact, as are all sums: below 2^53)
    double mine;   // its cost
    Request first; // its first request
    int run;
};
__device__ __forceinline__ double lane_of(double v, int lane) {
    const int2 u = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_readlane(u.x, lane), __builtin_amdgcn_readlane(u.y, lane)));
}
__device__ __forceinline__ double uniform(double v) { return lane_of(v, 0); }
__device__ __forceinline__ Line line_of(const TreeAttn& w) {
    const PagedAttnArgs& a = w.a;
    Line l;
    l.run = (a.n_req + 63) / 64;
    l.mine = 0.0;
    l.first = Request{0, 0, 0};
    float rows = 0.0f;
#pragma unroll 4
    for (int e = 0; e < l.run; e++) {
        const int r = (threadIdx.x & 63) * l.run + e;
        const Request q = request(a, min(r, a.n_req - 1));
        if (e == 0) l.first = q;
        l.mine += r < a.n_req ? shape_of(q, w.G).cost : 0.0;
        rows += r < a.n_req ? (float)q.n : 0.0f;
    }
    const double upto = scan64(l.mine);
    l.before = upto - l.mine;
    // row_starts that go up and down, so that requests overlap: nothing is done
    const bool overlap = wave_sum(rows) > 1.001f * (float)a.n_rows;
    const double total = overlap ? 0.0 : lane_of(upto, 63);
    l.cuts.pieces = uniform(total > 0.0 ? max(1, (int)fmin((double)w.blocks, total / kLeastPiece)) : 0);
    l.cuts.each = uniform(total / max(1, l.cuts.pieces));
    l.cuts.total = total;
    return l;
}

// A tile of a request, and its beginning counted from the request's.
struct Tile {
    int row0, rows, kind;  // kind: 128, 64 or 32 rows
    double at;
};
__device__ __forceinline__ Tile tile_of(const Shape& s, int tile) {
    Tile t;
    t.row0 = tile * kManyRows;
    t.at = tile * s.tile;
    t.rows = tile < s.whole ? kManyRows : s.rest;
    t.kind = t.rows > 64 ? 128 : t.rows > 32 ? 64 : 32;
    return t;
}
// The unit at which a cut `x` behind the tile's beginning divides it: 0 and `units` where it
// does not (near its ends, and where keys stay whole).
__device__ __forceinline__ int unit_at(const TreeAttn& w, double x, int units, int rows) {
    const int per = cost_of(rows);
    const int u = ((int)fmin(fmax(x, 0.0), (double)units * per + kCostTile) - kCostTile) / per;
    if (w.a.whole || u < kLeastUnits) return 0;
    return u > units - kLeastUnits ? units : u;
}

// The place of cut x (below the line's total).
__device__ __forceinline__ Place place_of(const TreeAttn& w, const Line& l, double x) {
    const uint64_t past = __ballot(l.before + l.mine > x);
    const int at = uniform(__ffsll((unsigned long long)past) - 1);
    double begin = lane_of(l.before, at);
    int r = at * l.run;
    Request q{__builtin_amdgcn_readlane(l.first.start, at), __builtin_amdgcn_readlane(l.first.n, at),
              __builtin_amdgcn_readlane(l.first.kv, at)};
    // the lane's run, 64 requests side by side
    for (int r0 = r; l.run > 1 && r0 < (at + 1) * l.run; r0 += 64) {
        const int mine = r0 + (threadIdx.x & 63);
        const Request of = request(w.a, min(mine, w.a.n_req - 1));
        const double cost = mine < min((at + 1) * l.run, w.a.n_req) ? shape_of(of, w.G).cost : 0.0, upto = scan64(cost);
        const uint64_t here = __ballot(begin + upto > x);
        if (here) {
            const int i = uniform(__ffsll((unsigned long long)here) - 1);
            r = r0 + i, begin += lane_of(upto - cost, i);
            q = Request{__builtin_amdgcn_readlane(of.start, i), __builtin_amdgcn_readlane(of.n, i), __builtin_amdgcn_readlane(of.kv, i)};
            break;
        }
        begin += lane_of(upto, 63);
    }
    const Shape s = shape_of(q, w.G);
    x -= begin;
    const int tiles = s.whole + s.rest_tiles, tile = tiles == 1 ? 0 : min(tiles - 1, (int)floor(x / s.tile));
    const Tile t = tile_of(s, tile);
    const int u = unit_at(w, x - t.at, s.units, t.rows);
    const bool next = u == s.units;
    return Place{uniform(r), uniform(next ? tile + 1 : tile), uniform(next ? 0 : u), uniform(begin), q};
}

// The first request behind r that has rows: lengths of 256 are requested together. (4 trees beside 252 idle slots
// 31 us, beside 2044 45; one slot at a time took 125 and 805. Of the 31 9 are the join, whose blocks are
// dealt out to as many tiles as requests could have.)
__device__ __forceinline__ int next_with_rows(const PagedAttnArgs& a, int r) {
    for (r++; r < a.n_req; r += 256) {
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) n[i] = request(a, min(r + 64 * i + ((int)threadIdx.x & 63), a.n_req - 1)).n;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t some = __ballot(n[i] > 0 && r + 64 * i + ((int)threadIdx.x & 63) < a.n_req);
            if (some) return r + 64 * i + __ffsll((unsigned long long)some) - 1;
        }
    }
    return a.n_req;
}

// A record holds results as the lanes have them: of 32 rows at a time and features 8 i .. + 7, the 4
// features of lane 32 h + row (h: 0 and 1) one after the other, so that a wave stores and loads 1 KB at
// once; behind them [record][2] maximum and sum.
template <int DH>
__device__ __forceinline__ int64_t in_record(int row, int feature) {
    return ((row >> 5) * (DH / 8) + (feature >> 3)) * 256 + ((feature >> 2) & 1) * 128 + (row & 31) * 4 + (feature & 3);
}

// A part of a tile's keys.
struct Segment {
    Request q;
    int r, row0, rows;
    int kb, ke;      // keys
    float* rec;      // nullptr: all of the tile's keys
};

// ---- tiles of 32 rows ------------------------------------------------------------------
// The four waves take the 32-key tiles in turn, each with its own buffers and no barrier:
// while a tile's scores become weights the next tile's keys are on their way, while its
// values are used the next values. The waves' results meet in LDS.
template <int DH, bool F16>
__device__ __forceinline__ void rows32(const TreeAttn& w, const Segment& g, int hk, uint8_t* lds, int tid) {
    constexpr int NW = 4, kTile = 32 * DH * 2, kLoads = kTile / 1024;
    __shared__ float2 s_ml[NW][32];
    __shared__ int s_bad[NW];
    __shared__ uint32_t s_again[NW];
    __shared__ int s_lim[32];  // the rows' reach within the part
    const PagedAttnArgs& a = w.a;
    const int G = w.G;
    const Request q = g.q;
    const int lane = tid & 63, h = lane >> 5, c32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int w0 = g.row0, n_rows = g.rows, kb = g.kb, ke = g.ke;
    const int row = w0 + min(c32, n_rows - 1);
    const int lim = min(ke, reach(a, q, row, G)), lim_lo = min(ke, seen_by_all(a, q, w0, G));
    if (tid < n_rows) s_lim[tid] = lim;
    auto sees_from = [&](int k) { return sees32(a, q, row, G, k, lim); };
    uint4 qf[DH / 16];
    load_q<DH>(a, q, row, hk, G, qf, lane);
    const float c = a.scale * kLog2e;
    floatx16 o[DH / 32];
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float m = ninf(), l = 0.0f;
    const int n_tiles = (max(0, ke - kb) + 31) / 32;
    const uint8_t *const kt = lds + wave * 2 * kTile, *const vt = kt + kTile;
    const uint32_t to = lds_addr(kt);
    // where the groups of the wave's next 16 tiles lie: lane 4 j + g holds group g of its tile j's
    const Filler<DH> fill(lane);
    int64_t where = 0;
    int bad_from = 0x7fffffff;
    auto look_up = [&](int t) {
        const int key = kb + (t + NW * (lane >> 2)) * 32 + (lane & 3) * 8;
        bool outside;
        where = key_at<DH>(a, g.r, hk, min(key, ke - 1), outside);
        if (outside && key < ke) bad_from = min(bad_from, key);
    };
    auto load = [&](auto v, int t, int j) {
        constexpr bool V = decltype(v)::value;
        const int k0 = kb + t * 32;
        const uint16_t* const pool = V ? a.v : a.k;
        const uint32_t at = to + (V ? kTile : 0);
        if (k0 + 32 <= ke) {
#pragma unroll
            for (int n = 0; n < 4; n++) fill.template fill<V, true, true>(pool, lane_of(where, 4 * j + n), n, at);
        } else {
#pragma unroll
            for (int n = 0; n < 4; n++)
                fill.template fill<V, false, true>(pool, lane_of(where, 4 * j + n), n, at, max(0, ke - 1 - (k0 + 8 * n)));
        }
    };
    using K = std::false_type;
    using Vals = std::true_type;
    if (wave < n_tiles) {
        look_up(wave);
        load(K{}, wave, 0);
        load(Vals{}, wave, 0);
    }
    int j = 0;
    for (int t = wave; t < n_tiles; t += NW) {
        const int k0 = kb + t * 32, next = t + NW, jn = (j + 1) & 15;
        const bool more = next < n_tiles, edge = k0 + 32 > lim_lo;
        wait_vmem<kLoads>();
        floatx16 s[1] = {scores32<DH, F16>(kt, qf, lane)};
        wait_lds();
        if (more) {
            if (jn == 0) look_up(next);
            load(K{}, next, jn);
        }
        weigh<1>(s, c, mask_and_move<DH, F16, true, 1>(s, k0, lim, edge, sees_from, c, m, l, o, lane), l);
        if (more) wait_vmem<kLoads>();
        else wait_vmem<0>();
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            uint32_t p[4][kTerms];
#pragma unroll
            for (int e = 0; e < 4; e++) split_pair<F16, kTerms>(s[0][8 * kk + 2 * e], s[0][8 * kk + 2 * e + 1], p[e]);
            values16<DH, F16>(vt + kk * 16 * 2 * DH, p, o, lane);
        }
        wait_lds();
        if (more) load(Vals{}, next, jn);
        j = jn;
    }
    l = pair32<false>(l);
    // the waves' results to LDS (their own buffers; the chunk of 4 features f of row c at f ^ c)
    const int bad = wave_min_int(bad_from);
    if (lane == 0) s_bad[wave] = bad;
    const uint32_t mine = rows_again<DH>(l, o, c32 < n_rows);
    if (lane == 0) s_again[wave] = mine;
    if (h == 0) s_ml[wave][c32] = make_float2(m, l);
    constexpr int kChunks = DH / 4;
    static_assert(32 * DH * 4 <= 2 * kTile, "a wave's results fit its buffers");
    if (c32 < n_rows)
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const int chunk = (8 * d + 2 * n + h) ^ (c32 & (kChunks - 1));
                *reinterpret_cast<float4*>(lds + wave * 2 * kTile + c32 * (DH * 4) + chunk * 16) =
                    make_float4(o[d][4 * n], o[d][4 * n + 1], o[d][4 * n + 2], o[d][4 * n + 3]);
            }
    __syncthreads();
    int bad_all = s_bad[0];
    uint32_t votes = s_again[0];
#pragma unroll
    for (int v = 1; v < NW; v++) bad_all = min(bad_all, s_bad[v]), votes |= s_again[v];
    float* const rec_ml = g.rec + w.record * DH;
    const uint32_t again = uniform((int)votes);
    if (again) {
        for (int x = wave; x < n_rows; x += NW) {
            if (!((again >> x) & 1u)) continue;
            float m1, l1, o1[DH / 64];
            const int rw = w0 + x, sees = uniform(s_lim[x]);
            row_again<DH, F16, true>(a, q, g.r, hk, hk * G + rw % G, q.start + rw / G, kb, sees, m1, l1, o1, lane);
            if (sees > bad_all) l1 = __builtin_nanf("");
            if (g.rec && lane == 0) *reinterpret_cast<float2*>(rec_ml + 2 * x) = make_float2(m1, l1);
#pragma unroll
            for (int e = 0; e < DH / 64; e++) {
                if (g.rec) g.rec[in_record<DH>(x, lane + 64 * e)] = o1[e];
                else store_out(a, out_at<DH>(a, q, rw, hk, G) + lane + 64 * e, sees ? o1[e] / l1 : 0.0f);
            }
        }
    }
    for (int i = tid; i < 32 * kChunks; i += 64 * NW) {
        // a record's 32 rows side by side, else a row's features
        const int x = g.rec ? i % 32 : i / kChunks, f = g.rec ? i / 32 : i % kChunks;
        if (x >= n_rows || ((again >> x) & 1u)) continue;
        float2 ml[NW];
        float mx = ninf();
#pragma unroll
        for (int v = 0; v < NW; v++) ml[v] = s_ml[v][x], mx = fmaxf(mx, ml[v].x);
        float sum = 0.0f, r0 = 0.0f, r1 = 0.0f, r2 = 0.0f, r3 = 0.0f;
#pragma unroll
        for (int v = 0; v < NW; v++) {
            if (v >= n_tiles) break;  // a wave without keys
            const float e = ml[v].x == mx ? 1.0f : __builtin_amdgcn_exp2f(ml[v].x - mx);
            const float4 y = *reinterpret_cast<const float4*>(lds + v * 2 * kTile + x * (DH * 4) +
                                                              (f ^ (x & (kChunks - 1))) * 16);
            sum = fmaf(ml[v].y, e, sum);
            r0 = fmaf(y.x, e, r0), r1 = fmaf(y.y, e, r1), r2 = fmaf(y.z, e, r2), r3 = fmaf(y.w, e, r3);
        }
        const int rw = w0 + x, sees = s_lim[x];
        if (sees > bad_all) sum = __builtin_nanf("");
        if (g.rec) {
            *reinterpret_cast<float4*>(g.rec + in_record<DH>(x, 4 * f)) = make_float4(r0, r1, r2, r3);
            if (f == 0) *reinterpret_cast<float2*>(rec_ml + 2 * x) = make_float2(mx, sum);
        } else {
            const float inv = sees ? 1.0f / sum : 0.0f;
            store_out4(a, out_at<DH>(a, q, rw, hk, G) + 4 * f, sees ? r0 * inv : 0.0f, sees ? r1 * inv : 0.0f,
                       sees ? r2 * inv : 0.0f, sees ? r3 * inv : 0.0f);
        }
    }
}

// ---- tiles of 64 and 128 rows ----------------------------------------------------------
// WR waves of 32 rows share tiles of 16 WR keys that they load together into two buffers:
// the next tile is on its way while one is used; one barrier a tile. With WR = 2 the block
// is two such groups that take the tiles in turn and join their results in LDS.
template <int DH, bool F16, int WR>
__device__ __forceinline__ void rows_shared(const TreeAttn& w, const Segment& g, int hk, uint8_t* lds, int tid) {
    constexpr int NW = 4, NG = NW / WR, TK = 64 / NG, kTile = TK * DH * 2, N = TK / 32;
    __shared__ int s_bad[NW];
    __shared__ float2 s_ml[64];
    const PagedAttnArgs& a = w.a;
    const int G = w.G;
    const Request q = g.q;
    const int lane = tid & 63, h = lane >> 5, c32 = lane & 31;
    const int all_waves = __builtin_amdgcn_readfirstlane(tid >> 6), group = all_waves / WR, wave = all_waves % WR;
    lds += group * 4 * kTile;
    const int last = g.row0 + g.rows, kb = g.kb, ke = g.ke;
    const int w0 = g.row0 + 32 * wave;  // the wave's first row
    const int row = min(w0 + c32, last - 1);
    const float c = a.scale * kLog2e;
    // the group's tiles, and the first group's (barriers are for all)
    const int n_all = (max(0, ke - kb) + TK - 1) / TK, n_tiles = max(0, (n_all - group + NG - 1) / NG), n_steps = (n_all + NG - 1) / NG;
    // the wave loads keys 16 wave .. + 15 of a tile; lane 2 j + n holds where its group n of tile j
    // of 32 lies, for keys and (a tile behind) for values
    const Filler<DH> fill(lane);
    int64_t where[2] = {0, 0};
    int bad_from = 0x7fffffff;
    auto load = [&](auto vals, int t) {
        constexpr bool V = decltype(vals)::value;
        if (t >= n_tiles) return;
        const int k0 = kb + (t * NG + group) * TK + 16 * wave;
        if ((t & 31) == 0 && (!V || t > 0)) {
            const int key = k0 + (lane >> 1) * (TK * NG) + (lane & 1) * 8;
            bool outside;
            where[V] = key_at<DH>(a, g.r, hk, min(key, ke - 1), outside);
            if (outside && key < ke) bad_from = min(bad_from, key);
        }
        const uint32_t to = lds_addr(lds) + ((t & 1) * 2 + V) * kTile + wave * (32 * DH);
        const uint16_t* const pool = V ? a.v : a.k;
        if (k0 + 16 <= ke) {
#pragma unroll
            for (int n = 0; n < 2; n++) fill.template fill<V, true, false>(pool, lane_of(where[V], 2 * (t & 31) + n), n, to);
        } else {
#pragma unroll
            for (int n = 0; n < 2; n++)
                fill.template fill<V, false, false>(pool, lane_of(where[V], 2 * (t & 31) + n), n, to,
                                             max(0, ke - 1 - (k0 + 8 * n)));
        }
    };
    using Keys = std::false_type;
    using Vals = std::true_type;
    auto meet = [&]() {
        wait_lds();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // A tile's scores are made while the one before it becomes weights: the products and the
    // exponentials do not depend on each other.
    constexpr int kLoads = 2 * (DH / 64);  // of a wave and tile
    load(Keys{}, 0);
    where[1] = where[0];
    load(Vals{}, 0);
    load(Keys{}, 1);
    // (the first keys and values are on their way)
    const int lim = min(ke, reach(a, q, row, G)), lim_lo = min(ke, seen_by_all(a, q, min(w0, last - 1), G));
    const int lim_hi = w0 < last ? min(ke, reach_of_tile(a, q, min(w0 + 31, last - 1), G)) : 0;
    auto sees_from = [&](int k) { return sees32(a, q, row, G, k, lim); };
    uint4 qf[DH / 16];
    load_q<DH>(a, q, row, hk, G, qf, lane);
    floatx16 o[DH / 32];
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float m = ninf(), l = 0.0f;
    if (n_tiles > 1) wait_vmem<2 * kLoads>();
    else wait_vmem<kLoads>();
    meet();
    auto scores = [&](const uint8_t* kt, floatx16 (&s)[N]) {
#pragma unroll
        for (int n = 0; n < N; n++) s[n] = scores32<DH, F16>(kt + n * 32 * 2 * DH, qf, lane);
    };
    auto step = [&](int t, floatx16 (&s)[N], floatx16 (&next)[N]) {
        const int k0 = kb + (t * NG + group) * TK;
        wait_vmem<0>();
        meet();  // this tile's values and the next one's keys are there, the last ones are used
        load(Vals{}, t + 1);
        load(Keys{}, t + 2);
        if (t >= n_tiles || k0 >= lim_hi) return;
        const uint8_t *const kt = lds + ((t + 1) & 1) * 2 * kTile, *const vt = lds + ((t & 1) * 2 + 1) * kTile;
        const float neg = mask_and_move<DH, F16, true, N>(s, k0, lim, k0 + TK > lim_lo, sees_from, c, m, l, o, lane);
        scores_and_weigh<DH, F16, N>(kt, qf, next, s, c, neg, l, lane);
        values<DH, F16, N>(vt, s, o, lane);
    };
    floatx16 s0[N], s1[N];
    scores(lds, s0);
    for (int t = 0; t < n_steps; t += 2) {
        step(t, s0, s1);
        if (t + 1 < n_steps) step(t + 1, s1, s0);
    }
    l = pair32<false>(l);
    const int bad = wave_min_int(bad_from);
    if (lane == 0) s_bad[all_waves] = bad;
    __syncthreads();
    int bad_all = s_bad[0];
#pragma unroll
    for (int v = 1; v < NW; v++) bad_all = min(bad_all, s_bad[v]);
    if constexpr (NG == 2) {
        // the second group's results, as its lanes hold them
        float4* const theirs = reinterpret_cast<float4*>(lds + (group ? 0 : 4 * kTile)) + wave * (8 * DH) + lane;
        if (group) {
#pragma unroll
            for (int d = 0; d < DH / 32; d++)
#pragma unroll
                for (int n = 0; n < 4; n++)
                    theirs[(4 * d + n) * 64] = make_float4(o[d][4 * n], o[d][4 * n + 1], o[d][4 * n + 2], o[d][4 * n + 3]);
            if (h == 0) s_ml[32 * wave + c32] = make_float2(m, l);
        }
        __syncthreads();
        if (group) return;
        const float2 ml = s_ml[32 * wave + c32];
        const float mx = fmaxf(m, ml.x);
        const float f0 = m == mx ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
        const float f1 = ml.x == mx ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mx);
        m = mx;
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float4 y = theirs[(4 * d + n) * 64];
                o[d][4 * n] = o[d][4 * n] * f0 + y.x * f1, o[d][4 * n + 1] = o[d][4 * n + 1] * f0 + y.y * f1;
                o[d][4 * n + 2] = o[d][4 * n + 2] * f0 + y.z * f1, o[d][4 * n + 3] = o[d][4 * n + 3] * f0 + y.w * f1;
            }
    }
    if (w0 >= last) return;
    float* const rec_ml = g.rec + w.record * DH;
    const uint32_t again = rows_again<DH>(l, o, w0 + c32 < last);
    if (again) {
        for (int x = 0; x < min(32, last - w0); x++) {
            if (!((again >> x) & 1u)) continue;
            float m1, l1, o1[DH / 64];
            const int rw = w0 + x, sees = min(ke, reach(a, q, rw, G)), y = 32 * wave + x;
            row_again<DH, F16, true>(a, q, g.r, hk, hk * G + rw % G, q.start + rw / G, kb, sees, m1, l1, o1, lane);
            if (sees > bad_all) l1 = __builtin_nanf("");
            if (g.rec && lane == 0) *reinterpret_cast<float2*>(rec_ml + 2 * y) = make_float2(m1, l1);
#pragma unroll
            for (int e = 0; e < DH / 64; e++) {
                if (g.rec) g.rec[in_record<DH>(y, lane + 64 * e)] = o1[e];
                else store_out(a, out_at<DH>(a, q, rw, hk, G) + lane + 64 * e, sees ? o1[e] / l1 : 0.0f);
            }
        }
    }
    if (w0 + c32 >= last || ((again >> c32) & 1u)) return;
    if (lim > bad_all) l = __builtin_nanf("");
    if (g.rec) {
        const int y = 32 * wave + c32;
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int n = 0; n < 4; n++)
                *reinterpret_cast<float4*>(g.rec + in_record<DH>(y, 32 * d + 8 * n + 4 * h)) =
                    make_float4(o[d][4 * n], o[d][4 * n + 1], o[d][4 * n + 2], o[d][4 * n + 3]);
        if (h == 0) *reinterpret_cast<float2*>(rec_ml + 2 * y) = make_float2(m, l);
        return;
    }
    const float inv = lim ? 1.0f / l : 0.0f;
    const int64_t at = out_at<DH>(a, q, row, hk, G);
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int n = 0; n < 4; n++)
            store_out4(a, at + 32 * d + 8 * n + 4 * h, o[d][4 * n] * inv, o[d][4 * n + 1] * inv, o[d][4 * n + 2] * inv,
                       o[d][4 * n + 3] * inv);
}

// The blocks that hold parts of the tile which cut j (1 .. pieces - 1) divides: the first one, and
// how many. x0: the tile's beginning on the line.
struct Parts {
    int first, count;
};
__device__ __forceinline__ Parts parts_of(const TreeAttn& w, const Cuts& l, int j, double x0, int units, int rows) {
    auto inside = [&](int i) {
        if (i < 1 || i >= l.pieces) return false;
        const int u = unit_at(w, l.at(i) - x0, units, rows);
        return u > 0 && u < units;
    };
    const int lane = threadIdx.x & 63;
    int from = j, to = j;  // the first and last cut inside
    for (;;) {
        const uint64_t out = __ballot(!inside(from - 1 - lane));
        from -= out ? __ffsll((unsigned long long)out) - 1 : 64;
        if (out) break;
    }
    for (;;) {
        const uint64_t out = __ballot(!inside(to + 1 + lane));
        to += out ? __ffsll((unsigned long long)out) - 1 : 64;
        if (out) break;
    }
    return Parts{uniform(from - 1), uniform(to - from + 2)};
}
// Where records lie, in floats: of the tile that goes on in a block, and of the one that begins there.
__device__ __forceinline__ int64_t record_at(const TreeAttn& w, int block, bool begins, int hk) {
    return ((int64_t)(begins ? w.blocks + block : block) * w.a.Hk + hk) * w.size;
}

// What a block keeps of its piece while it works on a tile (in LDS: the tiles need all registers).
struct Walk {
    Cuts cuts;
    Place at, end;
};

template <int DH, bool F16>
__global__ __launch_bounds__(256, DH == 256 ? 1 : 2) void tree_attn_kernel(TreeAttn w) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * 4 * 32 * DH * 2];  // 64 KB at a head_dim of 128
    __shared__ Walk s_walk;
    // (the grid's fastest axis: with 8 kv heads all blocks of a head share one XCD's L2)
    const int hk = blockIdx.x, b = blockIdx.y;
    {
        const Line l = line_of(w);
        if (b >= l.cuts.pieces) {
            if (w.split && hk == 0 && threadIdx.x == 0) w.split[b].at.x = 0;
            return;
        }
        const Place at = place_of(w, l, l.cuts.at(b));
        const Place end = b + 1 < l.cuts.pieces ? place_of(w, l, l.cuts.at(b + 1)) : Place{w.a.n_req, 0, 0, 0.0, Request{0, 0, 0}};
        if (threadIdx.x == 0) s_walk = Walk{l.cuts, at, end};
        if (w.split && hk == 0 && threadIdx.x == 0) w.split[b].at.x = 0;
    }
    for (;;) {
        // Thread 0's step at the loop's end is in LDS before the others read it. (The compiler leaves its own
        // wait out at this barrier, with which the loop begins: without this one, in one call of 64 requests of
        // 130 to 400, a wave went on from the place before and left wrong rows.)
        wait_lds();
        __syncthreads();
        const Place at = s_walk.at;
        const struct {
            int r, tile, unit;
        } p = {uniform(at.r), uniform(at.tile), uniform(at.unit)};
        const int end_r = uniform(s_walk.end.r), end_tile = uniform(s_walk.end.tile), end_unit = uniform(s_walk.end.unit);
        if (p.r > end_r || (p.r == end_r && (p.tile > end_tile || (p.tile == end_tile && p.unit >= end_unit)))) return;
        const Request q{uniform(at.q.start), uniform(at.q.n), uniform(at.q.kv)};
        const Shape s = shape_of(q, w.G);
        if (p.tile >= s.whole + s.rest_tiles) {
            if (at.begin + s.cost >= s_walk.cuts.total) return;  // the line's end
            const int r = uniform(next_with_rows(w.a, p.r));
            __syncthreads();
            if (threadIdx.x == 0) s_walk.at = Place{r, 0, 0, at.begin + s.cost, r < w.a.n_req ? request(w.a, r) : q};
            continue;
        }
        bool all;
        {
            const Tile t = tile_of(s, p.tile);
            const int to = p.r == end_r && p.tile == end_tile ? end_unit : s.units;
            all = p.unit == 0 && to == s.units;
            Segment g;
            g.q = q, g.r = p.r, g.row0 = t.row0, g.rows = t.rows;
            g.kb = p.unit * kUnit;
            g.ke = uniform(min(reach_of_tile(w.a, q, t.row0 + t.rows - 1, w.G), to * kUnit));
            g.rec = all ? nullptr : w.part + record_at(w, b, p.unit == 0, hk);
            int tid = threadIdx.x;
            asm volatile("" : "+v"(tid));  // (what a tile makes of it is not kept for the next: registers are short)
            if (t.kind == 32) rows32<DH, F16>(w, g, hk, lds, tid);
            else if (t.kind == 64) rows_shared<DH, F16, 2>(w, g, hk, lds, tid);
            else rows_shared<DH, F16, 4>(w, g, hk, lds, tid);
        }
        __syncthreads();
        if (!all && hk == 0 && w.split) {  // the joining launch learns of a tile from the block that it begins in
            const Place at = s_walk.at;
            const Request q{uniform(at.q.start), uniform(at.q.n), uniform(at.q.kv)};
            const Shape s = shape_of(q, w.G);
            const Tile t = tile_of(s, uniform(at.tile));
            const Parts parts = parts_of(w, s_walk.cuts, uniform(at.unit) > 0 ? b : b + 1, at.begin + t.at, s.units, t.rows);
            if (parts.first == b && threadIdx.x == 0) w.split[b] = Split{make_int4(parts.count, t.row0, t.rows, 0), make_int4(q.start, q.n, q.kv, 0)};
            __syncthreads();  // (all have read where the block is)
        }
        if (threadIdx.x == 0) s_walk.at.tile++, s_walk.at.unit = 0;
    }
}

// The parts of a cut tile joined in their order. Block y: the y-th such tile. An item is 8 features
// of 32 rows (in_record), 4 features of one row to a lane. A wave requests kJoin records of items
// together: 4 items of 2 parts, 2 of 4, one of more (64 requests of 20 to 60 tokens, some 500 tiles and 70 MB of
// records: 19 us, with one item at a time 25); beyond kJoin parts all four waves take a quarter of an item's parts each.
constexpr int kMergeWaves = 4, kJoin = 8;
template <int DH>
__global__ __launch_bounds__(64 * kMergeWaves) void tree_attn_merge_kernel(TreeAttn w) {
    __shared__ float s_sums[kMergeWaves][6][64];
    const PagedAttnArgs& a = w.a;
    const int hk = blockIdx.x, lane = threadIdx.x & 63, wave = (int)threadIdx.x / 64;
    // (a lane looks at two pieces, 128 are requested together)
    int left = blockIdx.y, b = -1;
    struct {
        int parts, row0, rows;
        Request q;
    } t;
    for (int b0 = 0; b0 < w.blocks && b < 0; b0 += 128) {
        Split mine[2];
#pragma unroll
        for (int i = 0; i < 2; i++) mine[i] = w.split[min(b0 + 64 * i + lane, w.blocks - 1)];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint64_t cut = __ballot(b0 + 64 * i + lane < w.blocks && mine[i].at.x > 0);
            const int count = __popcll(cut);
            if (b >= 0) continue;
            if (left >= count) {
                left -= count;
                continue;
            }
            for (; left > 0; left--) cut &= cut - 1;
            const int l = __ffsll((unsigned long long)cut) - 1;
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            b = b0 + 64 * i + l;
            t.parts = of(mine[i].at.x), t.row0 = of(mine[i].at.y), t.rows = of(mine[i].at.z);
            t.q = Request{of(mine[i].q.x), of(mine[i].q.y), of(mine[i].q.z)};
        }
    }
    if (b < 0) return;
    const int items = (t.rows + 31) / 32 * (DH / 8);
    struct Sums {
        float m, l, o[4];
        __device__ __forceinline__ void to(float top) {
            const float g = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
            m = top, l *= g, o[0] *= g, o[1] *= g, o[2] *= g, o[3] *= g;
        }
        __device__ __forceinline__ void join(float2 u, float4 y) {
            const float g = u.x == m ? 1.0f : __builtin_amdgcn_exp2f(u.x - m);
            l = fmaf(u.y, g, l);
            o[0] = fmaf(y.x, g, o[0]), o[1] = fmaf(y.y, g, o[1]);
            o[2] = fmaf(y.z, g, o[2]), o[3] = fmaf(y.w, g, o[3]);
        }
    };
    auto row_of = [&](int item) { return item / (DH / 8) * 32 + (lane & 31); };
    auto feature_of = [&](int item) { return item % (DH / 8) * 8 + (lane >> 5) * 4; };
    auto store = [&](int item, const Sums& s, bool sees) {
        const int x = row_of(item);
        if (item >= items || x >= t.rows) return;
        store_out4(a, out_at<DH>(a, t.q, t.row0 + x, hk, w.G) + feature_of(item), sees ? s.o[0] / s.l : 0.0f,
                   sees ? s.o[1] / s.l : 0.0f, sees ? s.o[2] / s.l : 0.0f, sees ? s.o[3] / s.l : 0.0f);
    };
    auto sees_any = [&](int item) { return reach(a, t.q, t.row0 + min(row_of(item), t.rows - 1), w.G) > 0; };
    // parts `from` on of I items, J parts together (rows behind the last: what their places hold is not stored)
    auto parts = [&](auto each, auto together, const int (&item)[decltype(each)::value], Sums (&s)[decltype(each)::value],
                     bool (&sees)[decltype(each)::value], int from, int to) {
        constexpr int I = decltype(each)::value, J = decltype(together)::value;
#pragma unroll
        for (int i = 0; i < I; i++) s[i] = Sums{ninf(), 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        for (int s0 = from; s0 < to; s0 += J) {
            float2 u[I * J];
            float4 y[I * J];
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int part = min(s0 + j, to - 1);
                const float* const rec = w.part + record_at(w, b + part, part == 0, hk);
#pragma unroll
                for (int i = 0; i < I; i++) {
                    const int x = row_of(item[i]);
                    u[I * j + i] = *reinterpret_cast<const float2*>(rec + w.record * DH + 2 * x);
                    y[I * j + i] = *reinterpret_cast<const float4*>(rec + in_record<DH>(x, feature_of(item[i])));
                }
            }
            if (s0 == from)
#pragma unroll
                for (int i = 0; i < I; i++) sees[i] = sees_any(item[i]);  // (the records are on their way)
#pragma unroll
            for (int i = 0; i < I; i++) {
                float top = s[i].m;
#pragma unroll
                for (int j = 0; j < J; j++) top = fmaxf(top, u[I * j + i].x);
                s[i].to(top);
#pragma unroll
                for (int j = 0; j < J; j++)
                    if (s0 + j < to) s[i].join(u[I * j + i], y[I * j + i]);
            }
        }
    };
    if (t.parts <= kJoin) {
        auto run = [&](auto each, auto together) {
            constexpr int I = decltype(each)::value;
            for (int item0 = (blockIdx.z * kMergeWaves + wave) * I; item0 < items; item0 += gridDim.z * kMergeWaves * I) {
                int item[I];
                bool sees[I];
                Sums s[I];
#pragma unroll
                for (int i = 0; i < I; i++) item[i] = min(item0 + i, items - 1);
                parts(each, together, item, s, sees, 0, t.parts);
#pragma unroll
                for (int i = 0; i < I; i++) store(item0 + i, s[i], sees[i]);
            }
        };
        if (t.parts <= 2) run(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
        else if (t.parts <= 4) run(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
        else run(std::integral_constant<int, 1>{}, std::integral_constant<int, kJoin>{});
        return;
    }
    const int each = (t.parts + kMergeWaves - 1) / kMergeWaves, from = min(t.parts, wave * each);
    for (int item = blockIdx.z; item < items; item += gridDim.z) {
        const int one[1] = {item};
        bool sees[1] = {false};
        Sums s[1];
        parts(std::integral_constant<int, 1>{}, std::integral_constant<int, kJoin>{}, one, s, sees, from, min(t.parts, from + each));
        __syncthreads();  // (the item before is read)
        float* const mine = &s_sums[wave][0][lane];
        mine[0] = s[0].m, mine[64] = s[0].l;
#pragma unroll
        for (int e = 0; e < 4; e++) mine[64 * (2 + e)] = s[0].o[e];
        __syncthreads();
        if (wave > 0) continue;
        float top = s[0].m;
#pragma unroll
        for (int v = 1; v < kMergeWaves; v++) top = fmaxf(top, s_sums[v][0][lane]);
        s[0].to(top);
#pragma unroll
        for (int v = 1; v < kMergeWaves; v++) {
            const float* const q = &s_sums[v][0][lane];
            s[0].join(make_float2(q[0], q[64]), make_float4(q[128], q[192], q[256], q[320]));
        }
        store(item, s[0], sees[0]);
    }
}

struct Launch {
    TreeAttn w;
    int cut, shares;  // most tiles that are cut, and the blocks that join one
    size_t records, bytes;
};
Launch plan_launch(const PagedAttnArgs& a, int num_cus) {
    Launch L{};
    const int64_t G = a.Hq / a.Hk, rows = (int64_t)a.n_rows * G;
    L.w.a = a;
    L.w.G = (int)G;
    // blocks resident at once (LDS and registers)
    const int64_t room = std::max<int64_t>(1, (int64_t)num_cus * (a.Dh == 256 ? 1 : 2) / a.Hk);
    L.w.blocks = (int)room;
    L.w.record = (int)(std::min<int64_t>(rows, kManyRows) + 31) / 32 * 32;
    L.w.size = (L.w.record * (a.Dh + 2) + 31) / 32 * 32;
    L.records = (size_t)2 * L.w.blocks * a.Hk * L.w.size * sizeof(float);
    L.bytes = L.w.blocks > 1 ? L.records + L.w.blocks * sizeof(Split) : 0;  // (a line in one piece: nothing is cut)
    const int64_t few = std::min<int64_t>((int64_t)a.max_new * G, rows);
    // tiles: a request's whole ones and one more; a cut divides one tile
    const int64_t tiles = std::min<int64_t>(a.n_req, a.n_rows) + rows / kManyRows;
    L.cut = (int)std::min<int64_t>(L.w.blocks - 1, tiles);
    // a block for every item (as the hint says), over about eight blocks to a CU
    const int64_t items = (std::min<int64_t>(std::max<int64_t>(few, 1), kManyRows) + 31) / 32 * (a.Dh / 8);
    L.shares = (int)std::max<int64_t>(1, std::min(items, 8 * (int64_t)num_cus / std::max<int64_t>(1, (int64_t)L.cut * a.Hk)));
    return L;
}

}  // namespace

size_t paged_tree_attn_workspace_bytes(const PagedAttnArgs& a, int num_cus) {
    return plan_launch(a, num_cus).bytes;
}

Status launch_paged_tree_attn(const PagedAttnArgs& a, void* workspace, size_t workspace_bytes, int num_cus, hipStream_t st) {
    Launch L = plan_launch(a, num_cus);
    if (!a.whole && L.bytes > workspace_bytes)
        return Status::fail(JH_ERR_INVALID, "jh_paged_tree_attention: the workspace does not hold the parts");
    L.w.part = static_cast<float*>(workspace);
    if (!a.whole && L.bytes) L.w.split = reinterpret_cast<Split*>(static_cast<char*>(workspace) + L.records);
    const dim3 grid((unsigned)a.Hk, (unsigned)L.w.blocks);
    auto with = [&](auto dh) {
        constexpr int DH = decltype(dh)::value;
        if (a.f16) hipLaunchKernelGGL((tree_attn_kernel<DH, true>), grid, dim3(256), 0, st, L.w);
        else hipLaunchKernelGGL((tree_attn_kernel<DH, false>), grid, dim3(256), 0, st, L.w);
        if (L.w.split && L.cut > 0)
            hipLaunchKernelGGL(tree_attn_merge_kernel<DH>, dim3((unsigned)a.Hk, (unsigned)L.cut, (unsigned)L.shares),
                               dim3(64 * kMergeWaves), 0, st, L.w);
    };
    if (a.Dh == 64) with(std::integral_constant<int, 64>{});
    else if (a.Dh == 128) with(std::integral_constant<int, 128>{});
    else with(std::integral_constant<int, 256>{});
    return Status::ok();
}

}  // namespace jh
