// Attention of every request's new tokens over a paged key/value cache (the rows of
// jh_paged_attention) on the matrix cores: o = softmax(scale q K^T) V with an online
// softmax, head_dim 64, 128 or 256, bf16 or f16.
//
// The rows of a kv head are its G query heads of each new token: row j of a request is
// head j % G of token j / G, so the heads that share keys and values read them once.
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T: a lane holds one row
// (lane % 32) of both accumulators, the row's maximum, sum and rescale are per-lane
// scalars, and the scores become the second product's B operand where they are. Its
// K order is the order the first product leaves the keys in, and the transposing LDS
// reads (ds_read_b64_tr_b16) take V in that order straight from its rows.
//
// Keys and values go to LDS by loads that need no registers (global_load_lds, 1 KB per
// wave and instruction, issued from inline asm with explicit waits): eight keys lie in
// one page, so a group's page is looked up once, its address is scalar, and the lanes
// add constants. 16-byte chunks are permuted within a row on the way (by the lanes'
// source addresses), so that neither kind of LDS read meets a bank conflict. Keys past
// the last one that a tile sees are loaded as that last one again: what lies in unused
// slots never enters.
//
// Work: a block takes a tile of rows of one request and kv head and a part of its keys.
// Lengths live on the device, so the blocks find their tile themselves, by running sums
// over the requests; the grid is the most that the sizes known to the host allow. Keys
// are split where that fills the GPU: all tiles' keys over about as many parts as blocks
// are resident, none so small that its records cost more than its keys. The parts of a
// tile are joined in their order: by a launch that follows, or, where rows are few and
// all blocks of a kv head run on one XCD (heads a multiple of 8), by the last of them.
//
// What bounds it, and figures on MI355X (calls in a row, their launches' gaps included;
// 32 query heads over 8 of 128 unless said):
//   few rows: HBM. 32 tokens of 8000 bf16 keys 167 us (6.3 TB/s), 64 of 100 to 8000
//     87 us (5.7), one of 100001 f16 keys over 4 heads 43 us (36 and 7 for the join). Loads are
//     non-temporal: 32 of 8000 take 189 us without. Short ones are chains of
//     round trips (lengths, tables, keys, records): 1 token of 64 keys 6 us, of 700 9 to 10;
//     with a launch of its own for the join 9 and 11 us.
//   many rows: 2000 tokens of 8000 bf16 keys 323 to 348 us, by device: 660 to 710 TFLOP/s
//     of the formula's operations, and, the second product being made twice (kTerms), 990
//     to 1050 of the matrix cores', where a large bf16 product of the library reaches 1180
//     to 1350. By counters the MFMA pipes are busy 52 % of the time at 1.8 GHz and VALU
//     47 %. Built with 256 registers. 513 tokens of 513 24 us, of which
//     4 are a merge launch that finds nothing to join: 136 blocks walk five steps of keys.
#include "paged_attention.hpp"

namespace jh {
namespace {

// Requests of up to this many rows take tiles of 32, which read keys once per tile but
// leave no wave idle: 16 runs of 2 to 7 tokens (8 rows each) 26.7 us, 32.5 with a limit of
// 32; a run beyond takes tiles of 128 (two pieces of prompts beside 22 tokens 42 us).
constexpr int kFewLimit = 64;

// ---- finding a block's work ---------------------------------------------------------
struct Attn {
    PagedAttnArgs a;
    int G;           // Hq / Hk
    double per_target;  // 1 / target
    int few;         // requests of at most this many rows (new tokens * G) take tiles of 32 rows, others of 128
    int target;      // parts of the keys to make, per kv head
    int record;      // rows of a record
    int size;        // floats of a record: whole 128-byte lines, so that no two XCDs write one
    int arrivals;    // of a kv head, in `sync` (whole lines too)
    int* sync;       // arrivals at [kv head][slot of a split tile's first record], zero between calls; nullptr: a
                     // merge launch joins the parts
    float* part;     // records of split parts: [record][DH] results, then [record][2] maximum and sum
};
// Least units of a part: two (a 32-key tile per wave), and one more for every kRowsPerUnit
// rows of results that a part writes and the merge reads.
constexpr int kLeast = 2, kRowsPerUnit = 21;

struct Work {
    bool ok;
    int r, local;     // the request, and the index among its items
    Request q;
    bool few;
    int tiles, splits, per;  // row tiles; parts of the keys, `per` units each
    int slot;         // of its first record
};

// The item `index` of all requests: tiles * splits items per request, or, with MERGE, the
// row tiles of requests whose keys are split. By every wave of a block for itself: a lane
// sums a run of requests, a scan over the lanes, and the run that holds the item is
// walked by all lanes together.
template <bool MERGE>
__device__ __forceinline__ Work find_work(const Attn& w, int index) {
    const PagedAttnArgs& a = w.a;
    const int lane = threadIdx.x & 63, G = w.G, run = (a.n_req + 63) / 64;
    auto tiles_of = [&](const Request& q) {
        const int rows = q.n * G;
        return rows <= w.few ? (rows + kFewRows - 1) / kFewRows : (rows + kManyRows - 1) / kManyRows;
    };
    auto units_of = [&](const Request& q) { return max(1, (q.kv + kUnit - 1) / kUnit); };
    double all = 0.0;  // exact: below 2^53
    float new_rows = 0.0f;
    Request mine{0, 0, 0};
    for (int e = 0; e < run; e++) {
        const int r = lane * run + e;
        if (r >= a.n_req) break;
        const Request q = request(a, r);
        if (e == 0) mine = q;
        new_rows += (float)q.n;
        all += (double)tiles_of(q) * (double)units_of(q);
    }
    // row_starts that go up and down, so that requests overlap: more items than the grid was
    // made for (it has room for 0.1 %), and nothing is done
    if (wave_sum(new_rows) > 1.001f * (float)a.n_rows) return Work{};
    all = scan64(all);
    const double total = __builtin_bit_cast(
        double, make_int2(__builtin_amdgcn_readlane(__builtin_bit_cast(int2, all).x, 63),
                          __builtin_amdgcn_readlane(__builtin_bit_cast(int2, all).y, 63)));
    // least units of a part that leave at most `target` of them
    const int most = a.whole ? 1 << 30 : (int)min(fma(total, w.per_target, 1.0), 1073741824.0);
    auto splits_of = [&](const Request& q) {
        const int rows = q.n * G, units = units_of(q);
        int each = max(most, kLeast + min(rows, rows <= w.few ? kFewRows : kManyRows) / kRowsPerUnit);  // units per part
        // joined by one block, a part costs about a ninth of a unit: least of C + units / C / 9
        if (w.sync) each = max(each, (int)sqrtf((float)units * (1.0f / 9.0f)));
        // (a rounded quotient: any count near it will do, the same in every block)
        return max(1, (int)((float)(units + each / 2) * __builtin_amdgcn_rcpf((float)each)));
    };
    int items = 0, slots = 0, my_tiles = 0, my_splits = 1;
    for (int e = 0; e < run; e++) {
        const int r = lane * run + e;
        if (r >= a.n_req) break;
        const Request q = e == 0 ? mine : request(a, r);
        const int t = tiles_of(q), s = splits_of(q);
        if (e == 0) my_tiles = t, my_splits = s;
        items += MERGE ? (s > 1 ? t : 0) : t * s;
        slots += s > 1 ? t * s : 0;
    }
    const int upto = scan64(items), slots_upto = scan64(slots);
    const uint64_t past = __ballot(upto > index);
    Work o{};
    if (!past) return o;
    const int at = uniform(__ffsll((unsigned long long)past) - 1);
    int left = index - __builtin_amdgcn_readlane(upto - items, at);
    int slot = __builtin_amdgcn_readlane(slots_upto - slots, at);
    for (int e = 0; e < run; e++) {
        const int r = at * run + e;
        if (r >= a.n_req) break;
        Request q;
        int t, s;
        if (e == 0) {
            t = __builtin_amdgcn_readlane(my_tiles, at);
            s = __builtin_amdgcn_readlane(my_splits, at);
            q.start = __builtin_amdgcn_readlane(mine.start, at);
            q.n = __builtin_amdgcn_readlane(mine.n, at);
            q.kv = __builtin_amdgcn_readlane(mine.kv, at);
        } else {
            q = request(a, r);
            t = tiles_of(q), s = splits_of(q);
        }
        const int count = MERGE ? (s > 1 ? t : 0) : t * s;
        if (left < count) {
            o.ok = true, o.r = uniform(r), o.local = uniform(left), o.tiles = uniform(t), o.splits = uniform(s);
            o.q = Request{uniform(q.start), uniform(q.n), uniform(q.kv)};
            o.few = o.q.n * G <= w.few;
            o.per = uniform((units_of(q) + s - 1) / s);
            o.slot = uniform(slot);
            return o;
        }
        left -= count;
        slot += s > 1 ? t * s : 0;
    }
    return o;
}

constexpr auto no_mask = [](int) { return 0u; };

// ---- joining the parts -----------------------------------------------------------------
// Rows of one tile of one kv head whose keys were split, `first`, first + stride, ...
// times the rows at once: groups of DH / 4 lanes, 4 features each, one to a row for every
// 8 parts (all requested together); a row's groups meet in LDS in their order. L2: the
// records were stored by this launch on this XCD (device-coherent loads: past the CU's L1).
constexpr int kJoinBatch = 8;
template <int DH, int NT, bool L2>
__device__ __forceinline__ void join_rows(const Attn& w, const Work& k, int hk, int tile, int parts, int first, int stride,
                                          float4* s_o, float2* s_ml) {
    constexpr int kLanes = DH / 4, kGroups = NT / kLanes, kBatch = kJoinBatch;
    const PagedAttnArgs& a = w.a;
    const int G = w.G, rows = k.q.n * G, tr = k.few ? kFewRows : kManyRows;
    const int64_t step = (int64_t)a.Hk * w.size;
    const float* const rec = w.part + ((int64_t)(k.slot + tile * k.splits) * a.Hk + hk) * w.size;
    const auto rsrc = make_rsrc(rec, 0x7FFFFFFFu);  // (L2: the launch keeps the records below 2^31 bytes)
    const int f = threadIdx.x % kLanes, group = threadIdx.x / kLanes, count = min(tr, rows - tile * tr);
    // groups to a row: for its parts, as long as the block's rows find room beside each other
    const int here = (count + stride - 1) / stride;
    int each = 1;
    while (each * kBatch < parts && 2 * each * here <= kGroups) each *= 2;
    const int sub = group % each, at_once = kGroups / each;
    for (int x0 = first * at_once; x0 < count; x0 += stride * at_once) {
        const int x = min(x0 + group / each, count - 1);
        // (a part without keys of the row: a maximum of -inf, a sum of 0)
        float mx = ninf(), l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s0 = sub; s0 < parts; s0 += each * kBatch) {
            float2 u[kBatch];
            float4 y[kBatch];
            float top = mx;
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const int64_t at = min(s0 + i * each, parts - 1) * step;
                if constexpr (L2) {
                    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
                    u[i] = __builtin_bit_cast(float2, (u32x2_t)__builtin_amdgcn_raw_buffer_load_b64(
                                                          rsrc, (uint32_t)(at + w.record * DH + 2 * x) * 4, 0, kAuxSc1));
                    y[i] = __builtin_bit_cast(float4, (u32x4_t)__builtin_amdgcn_raw_buffer_load_b128(
                                                          rsrc, (uint32_t)(at + x * DH + 4 * f) * 4, 0, kAuxSc1));
                } else {
                    u[i] = *reinterpret_cast<const float2*>(rec + at + (int64_t)w.record * DH + 2 * x);
                    y[i] = *reinterpret_cast<const float4*>(rec + at + (int64_t)x * DH + 4 * f);
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; i++) top = fmaxf(top, s0 + i * each < parts ? u[i].x : top);
            const float g0 = mx == top ? 1.0f : __builtin_amdgcn_exp2f(mx - top);
            l *= g0, o[0] *= g0, o[1] *= g0, o[2] *= g0, o[3] *= g0;
            mx = top;
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                if (s0 + i * each >= parts) break;
                const float g = u[i].x == mx ? 1.0f : __builtin_amdgcn_exp2f(u[i].x - mx);
                l = fmaf(u[i].y, g, l);
                o[0] = fmaf(y[i].x, g, o[0]), o[1] = fmaf(y[i].y, g, o[1]);
                o[2] = fmaf(y[i].z, g, o[2]), o[3] = fmaf(y[i].w, g, o[3]);
            }
        }
        if (each > 1) {
            __syncthreads();  // (the round before has read)
            s_o[group * kLanes + f] = make_float4(o[0], o[1], o[2], o[3]);
            if (f == 0) s_ml[group] = make_float2(mx, l);
            __syncthreads();
        }
        if (sub != 0 || x0 + group / each >= count) continue;
        for (int g = 1; g < each; g++) mx = fmaxf(mx, s_ml[group + g].x);
        if (each > 1) l = o[0] = o[1] = o[2] = o[3] = 0.0f;
        for (int g = 0; each > 1 && g < each; g++) {
            const float2 u = s_ml[group + g];
            const float4 y = s_o[(group + g) * kLanes + f];
            const float h = u.x == mx ? 1.0f : __builtin_amdgcn_exp2f(u.x - mx);
            l = fmaf(u.y, h, l);
            o[0] = fmaf(y.x, h, o[0]), o[1] = fmaf(y.y, h, o[1]), o[2] = fmaf(y.z, h, o[2]), o[3] = fmaf(y.w, h, o[3]);
        }
        const int row = tile * tr + x;
        const bool sees = seen(k.q, row, G) > 0;
        store_out4(a, out_at<DH>(a, k.q, row, hk, G) + 4 * f, sees ? o[0] / l : 0.0f, sees ? o[1] / l : 0.0f,
                   sees ? o[2] / l : 0.0f, sees ? o[3] / l : 0.0f);
    }
}

// ---- few rows ------------------------------------------------------------------------
// Tiles of 32 rows: decode (a token's G heads) and short runs of new tokens. The NW
// waves take the part's 32-key tiles in turn, each with its own buffers and no barrier:
// while a tile's scores become weights the next tile's keys are on their way, while its
// values are used the next values. The waves' results meet in LDS.
template <int DH, bool F16, int NW>
__device__ __forceinline__ void few_rows(const Attn& w, const Work& k, int hk, uint8_t* lds) {
    constexpr int kTile = 32 * DH * 2, kLoads = kTile / 1024;
    __shared__ float2 s_ml[NW][32];
    __shared__ int s_bad[NW];
    __shared__ uint32_t s_again[NW];
    const PagedAttnArgs& a = w.a;
    const int G = w.G;
    const int tile = uniform(k.local / k.splits), split = k.local - tile * k.splits;
    const Request q = k.q;
    const int lane = threadIdx.x & 63, h = lane >> 5, c32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w0 = tile * kFewRows, n_rows = min(kFewRows, q.n * G - w0);
    const int kb = split * k.per * kUnit;
    // keys this part ends at: for the tile's last row, this lane's row, the first row
    const int end = uniform(seen(q, w0 + n_rows - 1, G));
    const int parts = max(1, (end + k.per * kUnit - 1) / (k.per * kUnit));
    if (split >= parts) return;
    const int ke = min(end, kb + k.per * kUnit);
    const int row = w0 + min(c32, n_rows - 1);
    const int lim = min(ke, seen(q, row, G)), lim_lo = min(ke, seen(q, w0, G));
    uint4 qf[DH / 16];
    load_q<DH>(a, q, row, hk, G, qf);
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
    const Filler<DH> fill;
    int64_t where = 0;
    int bad_from = 0x7fffffff;
    auto look_up = [&](int t) {
        const int key = kb + (t + NW * (lane >> 2)) * 32 + (lane & 3) * 8;
        bool outside;
        where = key_at<DH>(a, k.r, hk, min(key, ke - 1), outside);
        if (outside && key < ke) bad_from = min(bad_from, key);
    };
    auto load = [&](auto v, int t, int j) {
        constexpr bool V = decltype(v)::value;
        const int k0 = kb + t * 32;
        const uint16_t* const pool = V ? a.v : a.k;
        const uint32_t at = to + (V ? kTile : 0);
        if (k0 + 32 <= ke) {
#pragma unroll
            for (int g = 0; g < 4; g++) fill.template fill<V, true, true>(pool, lane_of(where, 4 * j + g), g, at);
        } else {
#pragma unroll
            for (int g = 0; g < 4; g++)
                fill.template fill<V, false, true>(pool, lane_of(where, 4 * j + g), g, at, max(0, ke - 1 - (k0 + 8 * g)));
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
        floatx16 s[1] = {scores32<DH, F16>(kt, qf)};
        wait_lds();
        if (more) {
            if (jn == 0) look_up(next);
            load(K{}, next, jn);
        }
        weigh<1>(s, c, mask_and_move<DH, F16, false, 1>(s, k0, lim, edge, no_mask, c, m, l, o), l);
        if (more) wait_vmem<kLoads>();
        else wait_vmem<0>();
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            uint32_t p[4][kTerms];
#pragma unroll
            for (int e = 0; e < 4; e++) split_pair<F16, kTerms>(s[0][8 * kk + 2 * e], s[0][8 * kk + 2 * e + 1], p[e]);
            values16<DH, F16>(vt + kk * 16 * 2 * DH, p, o);
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
            for (int g = 0; g < 4; g++) {
                const int chunk = (8 * d + 2 * g + h) ^ (c32 & (kChunks - 1));
                *reinterpret_cast<float4*>(lds + wave * 2 * kTile + c32 * (DH * 4) + chunk * 16) =
                    make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
            }
    __syncthreads();
    int bad_all = s_bad[0];
    uint32_t votes = s_again[0];
#pragma unroll
    for (int v = 1; v < NW; v++) bad_all = min(bad_all, s_bad[v]), votes |= s_again[v];
    const int64_t slot = (int64_t)(k.slot + k.local) * a.Hk + hk;
    float *const rec = w.part + slot * w.size, *const rec_ml = rec + w.record * DH;
    const uint32_t again = uniform((int)votes);
    if (again) {
        for (int x = wave; x < n_rows; x += NW) {
            if (!((again >> x) & 1u)) continue;
            float m1, l1, o1[DH / 64];
            const int rw = w0 + x, sees = min(ke, seen(q, rw, G));
            row_again<DH, F16, false>(a, q, k.r, hk, hk * G + rw % G, q.start + rw / G, kb, sees, m1, l1, o1);
            if (sees > bad_all) l1 = __builtin_nanf("");
            if (parts > 1 && lane == 0) *reinterpret_cast<float2*>(rec_ml + 2 * x) = make_float2(m1, l1);
#pragma unroll
            for (int e = 0; e < DH / 64; e++) {
                if (parts > 1) rec[x * DH + lane + 64 * e] = o1[e];
                else store_out(a, out_at<DH>(a, q, rw, hk, G) + lane + 64 * e, sees ? o1[e] / l1 : 0.0f);
            }
        }
    }
    for (int i = threadIdx.x; i < n_rows * kChunks; i += 64 * NW) {
        const int x = i / kChunks, f = i % kChunks;
        if ((again >> x) & 1u) continue;
        float2 ml[NW];
        float mx = ninf();
#pragma unroll
        for (int v = 0; v < NW; v++) ml[v] = s_ml[v][x], mx = fmaxf(mx, ml[v].x);
        float sum = 0.0f, r0 = 0.0f, r1 = 0.0f, r2 = 0.0f, r3 = 0.0f;
#pragma unroll
        for (int v = 0; v < NW; v++) {
            const float g = ml[v].x == ninf() ? 0.0f : __builtin_amdgcn_exp2f(ml[v].x - mx);
            if (v >= n_tiles) break;  // a wave without keys
            const float4 y = *reinterpret_cast<const float4*>(lds + v * 2 * kTile + x * (DH * 4) +
                                                              (f ^ (x & (kChunks - 1))) * 16);
            sum = fmaf(ml[v].y, ml[v].x == mx ? 1.0f : g, sum);
            const float gg = ml[v].x == mx ? 1.0f : g;
            r0 = fmaf(y.x, gg, r0), r1 = fmaf(y.y, gg, r1), r2 = fmaf(y.z, gg, r2), r3 = fmaf(y.w, gg, r3);
        }
        const int rw = w0 + x, sees = min(ke, seen(q, rw, G));
        if (sees > bad_all) sum = __builtin_nanf("");
        if (parts > 1) {
            *reinterpret_cast<float4*>(rec + x * DH + 4 * f) = make_float4(r0, r1, r2, r3);
            if (f == 0) *reinterpret_cast<float2*>(rec_ml + 2 * x) = make_float2(mx, sum);
        } else if (sees) {
            store_out4(a, out_at<DH>(a, q, rw, hk, G) + 4 * f, r0 / sum, r1 / sum, r2 / sum, r3 / sum);
        } else {
            store_out4(a, out_at<DH>(a, q, rw, hk, G) + 4 * f, 0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    if (!w.sync || parts == 1) return;
    // The part that arrives last joins them. All parts of a kv head run on one XCD (the grid
    // deals head h to XCD h % 8) and meet in its L2: the records' stores are done before the
    // arrival is counted there, and are read past this CU's L1 after it.
    __shared__ int s_last;
    wait_vmem<0>();
    __syncthreads();
    int* const arrivals = w.sync + hk * w.arrivals + k.slot + tile * k.splits;
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(arrivals, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    __syncthreads();
    if (!s_last) return;
    join_rows<DH, 64 * NW, true>(w, k, hk, tile, parts, 0, 1, reinterpret_cast<float4*>(lds), &s_ml[0][0]);
    if (threadIdx.x == 0) __hip_atomic_store(arrivals, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- many rows -----------------------------------------------------------------------
// Tiles of 128 rows, 32 a wave, over 64-key tiles that four waves load together into two
// buffers: the next tile is on its way while one is used; one barrier a tile. Eight waves
// are two such groups that take the tiles in turn and join their results in LDS: where a
// CU has one tile of rows only, its keys are walked in half the time.
template <int DH, bool F16, int NW>
__device__ __forceinline__ void many_rows(const Attn& w, const Work& k, int hk, uint8_t* lds) {
    constexpr int kTile = 64 * DH * 2;
    constexpr int NG = NW / 4;
    __shared__ int s_bad[NW];
    __shared__ float2 s_ml[128];
    const PagedAttnArgs& a = w.a;
    const int G = w.G;
    // the last tiles (the longest) first
    const int up = uniform(k.local / k.splits), tile = k.tiles - 1 - up, split = k.local - up * k.splits;
    const Request q = k.q;
    const int lane = threadIdx.x & 63, h = lane >> 5, c32 = lane & 31;
    const int all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = all_waves / 4, wave = all_waves & 3;
    lds += group * 4 * kTile;
    const int rows = q.n * G, kb = split * k.per * kUnit;
    const int end = uniform(seen(q, min(rows, (tile + 1) * kManyRows) - 1, G));
    const int parts = max(1, (end + k.per * kUnit - 1) / (k.per * kUnit));
    if (split >= parts) return;
    const int ke = min(end, kb + k.per * kUnit);
    const int w0 = tile * kManyRows + 32 * wave;  // the wave's first row
    const int row = min(w0 + c32, rows - 1);
    const int lim = min(ke, seen(q, row, G)), lim_lo = min(ke, seen(q, min(w0, rows - 1), G));
    const int lim_hi = w0 < rows ? min(ke, seen(q, min(w0 + 31, rows - 1), G)) : 0;
    uint4 qf[DH / 16];
    load_q<DH>(a, q, row, hk, G, qf);
    const float c = a.scale * kLog2e;
    floatx16 o[DH / 32];
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float m = ninf(), l = 0.0f;
    // the group's tiles, and the first group's (barriers are for all)
    const int n_all = (max(0, ke - kb) + 63) / 64, n_tiles = max(0, (n_all - group + NG - 1) / NG), n_steps = (n_all + NG - 1) / NG;
    // the wave loads keys 16 wave .. + 15 of a tile; lane 2 j + g holds where its group g of tile j
    // of 32 lies, for keys and (a tile behind) for values
    const Filler<DH> fill;
    int64_t where[2] = {0, 0};
    int bad_from = 0x7fffffff;
    auto load = [&](auto vals, int t) {
        constexpr bool V = decltype(vals)::value;
        if (t >= n_tiles) return;
        const int k0 = kb + (t * NG + group) * 64 + 16 * wave;
        if ((t & 31) == 0 && (!V || t > 0)) {
            const int key = k0 + (lane >> 1) * (64 * NG) + (lane & 1) * 8;
            bool outside;
            where[V] = key_at<DH>(a, k.r, hk, min(key, ke - 1), outside);
            if (outside && key < ke) bad_from = min(bad_from, key);
        }
        const uint32_t to = lds_addr(lds) + ((t & 1) * 2 + V) * kTile + wave * (32 * DH);
        const uint16_t* const pool = V ? a.v : a.k;
        if (k0 + 16 <= ke) {
#pragma unroll
            for (int g = 0; g < 2; g++) fill.template fill<V, true, false>(pool, lane_of(where[V], 2 * (t & 31) + g), g, to);
        } else {
#pragma unroll
            for (int g = 0; g < 2; g++)
                fill.template fill<V, false, false>(pool, lane_of(where[V], 2 * (t & 31) + g), g, to,
                                             max(0, ke - 1 - (k0 + 8 * g)));
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
    if (n_tiles > 1) wait_vmem<2 * kLoads>();
    else wait_vmem<kLoads>();
    meet();
    auto step = [&](int t, floatx16 (&s)[2], floatx16 (&next)[2]) {
        const int k0 = kb + (t * NG + group) * 64;
        wait_vmem<0>();
        meet();  // this tile's values and the next one's keys are there, the last ones are used
        load(Vals{}, t + 1);
        load(Keys{}, t + 2);
        if (t >= n_tiles || k0 >= lim_hi) return;
        const uint8_t *const kt = lds + ((t + 1) & 1) * 2 * kTile, *const vt = lds + ((t & 1) * 2 + 1) * kTile;
        const float neg = mask_and_move<DH, F16, false, 2>(s, k0, lim, k0 + 64 > lim_lo, no_mask, c, m, l, o);
        // In the source's order where four waves walk 128 rows of a head_dim of 128 or more (2000 tokens of
        // 8000: 323 us, 339 in the compiler's); not with eight waves (22 tokens and two prompts' pieces 39.8
        // and 40.9) or a head_dim of 64 (2000 of 8000 208 and 209).
        if constexpr (NW == 4 && DH >= 128) {
            scores_and_weigh<DH, F16, 2>(kt, qf, next, s, c, neg, l, lane);
            values<DH, F16, 2>(vt, s, o, lane);
        } else {
            next[0] = scores32<DH, F16>(kt, qf);
            next[1] = scores32<DH, F16>(kt + 32 * 2 * DH, qf);
            weigh<2>(s, c, neg, l);
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
                uint32_t p[4][kTerms];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    split_pair<F16, kTerms>(s[kk >> 1][8 * (kk & 1) + 2 * e], s[kk >> 1][8 * (kk & 1) + 2 * e + 1], p[e]);
                values16<DH, F16>(vt + kk * 16 * 2 * DH, p, o);
            }
        }
    };
    floatx16 s0[2] = {scores32<DH, F16>(lds, qf), scores32<DH, F16>(lds + 32 * 2 * DH, qf)}, s1[2];
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
                for (int g = 0; g < 4; g++)
                    theirs[(4 * d + g) * 64] = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
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
            for (int g = 0; g < 4; g++) {
                const float4 y = theirs[(4 * d + g) * 64];
                o[d][4 * g] = o[d][4 * g] * f0 + y.x * f1, o[d][4 * g + 1] = o[d][4 * g + 1] * f0 + y.y * f1;
                o[d][4 * g + 2] = o[d][4 * g + 2] * f0 + y.z * f1, o[d][4 * g + 3] = o[d][4 * g + 3] * f0 + y.w * f1;
            }
    }
    const int64_t slot = (int64_t)(k.slot + tile * k.splits + split) * a.Hk + hk;
    float *const rec = w.part + slot * w.size, *const rec_ml = rec + w.record * DH;
    if (w0 >= rows) return;
    const uint32_t again = rows_again<DH>(l, o, w0 + c32 < rows);
    if (again) {
        for (int x = 0; x < min(32, rows - w0); x++) {
            if (!((again >> x) & 1u)) continue;
            float m1, l1, o1[DH / 64];
            const int rw = w0 + x, sees = min(ke, seen(q, rw, G)), y = 32 * wave + x;
            row_again<DH, F16, false>(a, q, k.r, hk, hk * G + rw % G, q.start + rw / G, kb, sees, m1, l1, o1);
            if (sees > bad_all) l1 = __builtin_nanf("");
            if (parts > 1 && lane == 0) *reinterpret_cast<float2*>(rec_ml + 2 * y) = make_float2(m1, l1);
#pragma unroll
            for (int e = 0; e < DH / 64; e++) {
                if (parts > 1) rec[y * DH + lane + 64 * e] = o1[e];
                else store_out(a, out_at<DH>(a, q, rw, hk, G) + lane + 64 * e, sees ? o1[e] / l1 : 0.0f);
            }
        }
    }
    if (w0 + c32 >= rows || ((again >> c32) & 1u)) return;
    if (lim > bad_all) l = __builtin_nanf("");
    if (parts > 1) {
        const int y = 32 * wave + c32;
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<float4*>(rec + y * DH + 32 * d + 8 * g + 4 * h) =
                    make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
        if (h == 0) *reinterpret_cast<float2*>(rec_ml + 2 * y) = make_float2(m, l);
        return;
    }
    const float inv = lim ? 1.0f / l : 0.0f;
    const int64_t at = out_at<DH>(a, q, row, hk, G);
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            store_out4(a, at + 32 * d + 8 * g + 4 * h, o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv,
                       o[d][4 * g + 3] * inv);
}

// MIXED: tiles of 128 rows and of 32; else of 32 alone.
template <int DH, bool F16, bool MIXED, int NW>
__global__ __launch_bounds__(64 * NW, DH == 256 || NW == 8 ? 1 : 2) void paged_attn_kernel(Attn w) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * NW * 32 * DH * 2];  // of either: 16 KB a wave at a head_dim of 128
    // (the grid's fastest axis: with 8 kv heads all tiles of a head share one XCD's L2)
    const int hk = blockIdx.x;
    const Work k = find_work<false>(w, blockIdx.z * gridDim.y + blockIdx.y);
    if (!k.ok) return;
    if constexpr (MIXED)
        if (!k.few) {
            many_rows<DH, F16, NW>(w, k, hk, lds);
            return;
        }
    few_rows<DH, F16, NW>(w, k, hk, lds);
}

constexpr int kMergeThreads = 512;
template <int DH>
__global__ __launch_bounds__(kMergeThreads) void paged_attn_merge_kernel(Attn w) {
    __shared__ float4 s_o[kMergeThreads];
    __shared__ float2 s_ml[kMergeThreads / (DH / 4)];
    const int hk = blockIdx.x, G = w.G;
    const Work k = find_work<true>(w, blockIdx.y);
    if (!k.ok) return;
    const int tile = k.local, tr = k.few ? kFewRows : kManyRows;
    const int end = uniform(seen(k.q, min(k.q.n * G, (tile + 1) * tr) - 1, G));
    const int parts = max(1, (end + k.per * kUnit - 1) / (k.per * kUnit));
    if (parts > 1) join_rows<DH, kMergeThreads, false>(w, k, hk, tile, parts, blockIdx.z, gridDim.z, s_o, s_ml);
}

// A call's tiles and grid. `max_new` is a hint: with at most 32 rows per request as it
// says (64 where the parts are joined in the launch), every request takes tiles of 32
// rows; else those of more than kFewLimit rows take tiles of 128. Runs of 2 to 7 tokens of
// 8 heads: with a merge launch 16 of them 26.8 us in blocks made for both tiles, 29.0 in
// blocks for tiles of 32; joined in the launch 64 of them 64 and 59, but 16 of 500 to 5000
// keys 40 and 49. `wide`: blocks of eight waves where that many still find a CU each (mixed
// lengths 42.5 us, 53 without; a prompt of 64 tokens loses 1.5 us, of 128 1.0, of 256 0.3,
// of 1024 nothing). `parts`: with few tiles so many that all blocks are resident at once,
// with many twice the room (64 of 100-8000: 87.9 us, 92.5 with the room alone, 88.1 with
// three times); for long runs, whose records are large, fewer (2000 of 8000 348 us, 351
// with the room, 395 with twice; a prompt of 1024 41, 47 and 47).
struct Launch {
    Attn w;
    bool only_few, wide;  // wide: blocks of eight waves
    int items, merges, merge_rows;  // blocks per kv head; blocks to a joined tile
    size_t bytes;
};

Launch plan_launch(const PagedAttnArgs& a, int num_cus, int* sync) {
    const int64_t G = a.Hq / a.Hk, rows = (int64_t)a.n_rows * G, requests = std::min(a.n_req, a.n_rows);
    Launch L{};
    // (heads dealt to the XCDs in turn)
    const bool join = sync && !a.whole && a.Hk % 8 == 0;
    L.only_few = std::min((int64_t)a.max_new * G, rows) <= (join ? kFewLimit : kFewRows);
    L.w.a = a;
    L.w.G = (int)G;
    L.w.few = L.only_few ? 0x7fffffff : kFewLimit;
    const int64_t full = rows / (L.only_few ? kFewRows : kManyRows), about = requests + full;
    // at most: a request of few rows may have a second tile, and overlapping rows (0.1 %)
    const int64_t tiles = about + (L.only_few ? 0 : std::min(requests, rows / (kFewRows + 1))) + full / 512;
    L.wide = !L.only_few && a.Dh != 256 && about * a.Hk <= num_cus;
    // blocks resident at once (LDS; at a head_dim of 64 registers), per kv head
    const int per_cu = a.Dh == 256 || L.wide ? 1 : a.Dh == 128 ? 2 : L.only_few ? 4 : 3;
    const int64_t room = std::max<int64_t>(1, num_cus * per_cu / a.Hk);
    const int64_t parts = L.only_few ? (2 * about <= room ? room - about : 2 * room)
                                     : std::max((room + 1) / 2, room - about / 2);
    L.w.target = (int)std::max<int64_t>(1, parts);
    L.w.per_target = 1.0 / L.w.target;
    L.w.record = (int)(std::min<int64_t>(rows, L.only_few ? kFewRows : kManyRows) + 3) / 4 * 4;  // whole 16 bytes
    // a request of t tiles of u units has u / C parts, rounded, at least one, and all t * u / C
    // together are at most `target`: items are at most `target` and one for each tile,
    // parts of split requests (u / C from 3/2 on) at most 4/3 `target`
    L.items = (int)(L.w.target + tiles);
    L.merges = (int)std::min<int64_t>(L.w.target, tiles);
    // rows of a tile (as the hint says) times the groups that an average request's parts want
    const int64_t mr = std::min<int64_t>(std::max(a.max_new, 1) * G, L.only_few ? kFewRows : kManyRows);
    const int64_t groups = kMergeThreads / (a.Dh / 4), want = (L.w.target / tiles + kJoinBatch - 1) / kJoinBatch;
    L.merge_rows = (int)std::max<int64_t>(1, (mr * std::max<int64_t>(1, std::min(want, groups)) + groups - 1) / groups);
    L.w.size = (L.w.record * (a.Dh + 2) + 31) / 32 * 32;
    L.w.arrivals = (2 * L.w.target + 31) / 32 * 32;
    L.bytes = (size_t)2 * L.w.target * a.Hk * L.w.size * sizeof(float);
    if (join && L.only_few && (int64_t)L.w.arrivals * a.Hk <= kPagedSyncSlots && L.bytes < (1u << 31)) L.w.sync = sync;
    return L;
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnArgs& a, int num_cus, int* sync) {
    return plan_launch(a, num_cus, sync).bytes;
}

Status launch_paged_attn(const PagedAttnArgs& a, void* workspace, size_t workspace_bytes, int num_cus, int* sync,
                         hipStream_t st) {
    Launch L = plan_launch(a, num_cus, sync);
    if (!a.whole && L.bytes > workspace_bytes)
        return Status::fail(JH_ERR_INVALID, "jh_paged_attention: the workspace does not hold the parts");
    L.w.part = static_cast<float*>(workspace);
    // heads fastest: block b takes kv head b % Hk; z: items past 2^15, and a merge's shares of rows
    auto go = [&](auto kernel, int64_t items, int shares, int threads) {
        const int64_t y = std::min<int64_t>(items, 1 << 15);
        const dim3 grid((unsigned)a.Hk, (unsigned)y, (unsigned)(shares ? shares : (items + y - 1) / y));
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, L.w);
    };
    auto with = [&](auto dh, auto f16) {
        constexpr int DH = decltype(dh)::value;
        constexpr bool F16 = decltype(f16)::value;
        if (L.only_few) go(paged_attn_kernel<DH, F16, false, 4>, L.items, 0, 256);
        else if (!L.wide) go(paged_attn_kernel<DH, F16, true, 4>, L.items, 0, 256);
        if constexpr (DH != 256)  // (its tiles fill the LDS)
            if (L.wide) go(paged_attn_kernel<DH, F16, true, 8>, L.items, 0, 512);
        if (!L.w.sync && !a.whole) go(paged_attn_merge_kernel<DH>, L.merges, L.merge_rows, kMergeThreads);
    };
    auto typed = [&](auto dh) { a.f16 ? with(dh, std::true_type{}) : with(dh, std::false_type{}); };
    if (a.Dh == 64) typed(std::integral_constant<int, 64>{});
    else if (a.Dh == 128) typed(std::integral_constant<int, 128>{});
    else typed(std::integral_constant<int, 256>{});
    return Status::ok();
}

}  // namespace jh
