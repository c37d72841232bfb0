// kv_shared.hip — attention of sequences in groups that share a prefix of the key/value cache.
//
// Mathematics.  The rows of a group (new tokens x query heads of a key head) all see all of the
// group's prefix, so over it they are the rows of one sequence, whose codes are read and
// turned once for all of them.  Over what stands behind the prefix every sequence is on its own.  Both
// passes are the kernels of kv_attend.h; of each a row has parts (maximum, sum, sums of values),
// and as softmax does not care in what order its sums are taken, joining all of them is the
// attention over all tokens:  m = max m_p, l = sum 2^(m_p - m) l_p, o = sum 2^(m_p - m) o_p / l.
#include "kv_attend.h"

#include <cmath>

namespace jhq {
namespace {

// What a pass keeps of its rows.  A worker has steps of 64 tokens of consecutive tiles (rows of one head of a
// sequence, tile of them at most).  A tile's steps are numbered from its `start` on: what comes before stands
// for what beginning a tile costs, so that workers that begin several end with the others (64 single
// tokens behind 16003: 72.3 us without, 66.8 with).  A tile of whose steps a worker has all is kept by
// its rows' places in the output (`whole`); of the two that it may begin or end in the middle of, in slot
// 2 worker (begun before it) and 2 worker + 1 (goes on after it).  Sums of values first, then maxima and
// sums.  joins: the worker that begins a tile, and how many more have parts of it.
struct Kept {
    float* slots;
    int64_t n;     // of them
    int tile, start;
    int2* joins;
    float* whole;
    int64_t rows;  // new tokens x query heads
};

__host__ __device__ inline int64_t even4(int64_t floats) { return (floats + 3) / 4 * 4; }

// Its floats, laid out from base on.
inline int64_t lay_out(Kept& k, float* base, int D, int64_t slots, int tile, int64_t joins, int64_t rows) {
    k.n = slots;
    k.tile = tile;
    k.rows = rows;
    k.slots = base;
    const int64_t j = slots * tile * (D + 2);
    k.joins = reinterpret_cast<int2*>(base + j);
    const int64_t w = j + even4(2 * joins);
    k.whole = base + w;
    return w + even4(rows * (D + 2));
}

// The number of a sequence's first tile: a sequence of q rows has q / tile + 1 at most.
__device__ inline int64_t first_tile(const Kept& k, const KvSeq& s, int seq, int G) {
    return s.row * G / k.tile + seq;
}

// Keeps a wave's rows from r0 on; slot -1: all of their tokens.
template <int BITS, int D, int NC>
__device__ inline void keep_part(const Kept& k, int64_t slot, const Share& w, const KvAttend& a, int r0,
                                 int lane, const Rows<BITS, D, NC>& r) {
    const int g = lane >> 4;
    float* const base = slot < 0 ? k.whole : k.slots;
    float* const ml = base + (slot < 0 ? k.rows : k.n * k.tile) * D;
#pragma unroll
    for (int x = 0; x < NC; x++) {
        const int row = r0 + x * 16 + (lane & 15);
        if (row >= w.r0 + w.rn) continue;
        int64_t q;
        const int64_t at = slot < 0 ? row_of(w, a, row, &q) : slot * k.tile + (row - w.r0);
#pragma unroll
        for (int t = 0; t < D / 16; t++)
            *reinterpret_cast<f4*>(base + at * D + t * 16 + g * 4) = r.o[x][t];
        if (g == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(r.m[x], r.l[x]);
    }
}

// Tokens that a sequence's rows see in a pass, and their steps.
__device__ inline int extent(const KvOwn&, const KvSeq& s, const KvAttend& a, int* lo, int* hi) {
    return steps_of(s, a, lo, hi);
}
__device__ inline int extent(const KvLead&, const KvSeq& s, const KvAttend&, int* lo, int* hi) {
    *lo = 0;
    *hi = s.q ? s.n : 0;
    return (*hi + kStep - 1) / kStep;
}

// Numbers of the steps of a head of a sequence.
template <class B>
__device__ inline int tile_steps(const B& b, const KvSeq& s, const KvAttend& a, const Kept& k) {
    int lo, hi;
    const int n = extent(b, s, a, &lo, &hi);
    return n ? (n + k.start) * ((s.q * a.G + k.tile - 1) / k.tile) : 0;
}

// A worker's way through its steps: f(w, slot) for each tile that it has steps of, in the order of
// sequences, heads, tiles.
template <class B, class F>
__device__ inline void each_tile(const KvCache& c, const B& b, const KvAttend& a, const Kept& k, int total,
                                 int workers, int least, int worker, int lane, bool first_lane, F f) {
    auto steps = [&](const KvSeq& s) { return tile_steps(b, s, a, k); };
    // Loaded anew: kept from both passes' sums, the lane's sequences cost registers (heads of 64 in 4 bits spill
    // 10 in the place of 6).
    const KvSeq s0 = lane_seq(c, b, lane);
    const Cut cut = cut_at(c, b, Total{total, steps(s0), s0}, max(least, (total + workers - 1) / workers), worker,
                           lane, steps);
    int at = cut.at;
    if (at >= cut.end) return;
    Share w;
    w.seq = cut.seq;
    w.s = cut.s;
    w.split = 0;
    w.any = true;
    w.alone = false;
    int lo, hi, n = extent(b, w.s, a, &lo, &hi) + k.start;
    int tiles = (w.s.q * a.G + k.tile - 1) / k.tile;
    w.head = (at - cut.first) / (n * tiles);
    int tile = (at - cut.first) % (n * tiles) / n, from = (at - cut.first) % n;
    while (true) {
        const int to = min(n, from + (cut.end - at));
        const bool begins = from <= k.start;
        if (to > k.start) {
            if (begins && first_lane)
                k.joins[(first_tile(k, w.s, w.seq, a.G) + tile) * c.H + w.head] =
                    int2{worker, (at + n - from - 1) / cut.per - worker};
            if (w.s.ok) {
                w.r0 = tile * k.tile;
                w.rn = min(k.tile, w.s.q * a.G - w.r0);
                span_of(w, a);
                w.lo = lo + (max(from, k.start) - k.start) * kStep;
                w.hi = min(w.hi, lo + (to - k.start) * kStep);
                f(w, begins && to == n ? int64_t(-1) : static_cast<int64_t>(2 * worker + begins));
            }
        }
        at += to - from;
        if (at >= cut.end) return;
        from = 0;
        if (++tile < tiles) continue;
        tile = 0;
        if (++w.head < c.H) continue;
        w.head = 0;
        do {
            w.s = kv_seq(b, ++w.seq, c.shift);
            n = extent(b, w.s, a, &lo, &hi);
            tiles = n ? (w.s.q * a.G + k.tile - 1) / k.tile : 0;
            n += k.start;
        } while (tiles == 0);
    }
}

// One wave's steps of few rows (16 NT at most), straight from the cache into registers; sc: 192
// floats of LDS, the wave's.
template <int BITS, int D, int NT, class B>
__device__ inline void few_steps(const KvCache& c, const B& b, const KvAttend& a, const Kept& k, int total,
                                 int workers, int worker, int lane, float* sc) {
    each_tile(c, b, a, k, total, workers, kLeast, worker, lane, lane == 0, [&](const Share& w, int64_t slot) {
        Rows<BITS, D, NT> rows;
        Stream<BITS, D, NT> st(c, b, w, lane);
        rows.start(w, a, 0, lane);
        st.open(w.lo, kStep);
        float own[NT];
        const float big = rows.largest(a, own);
        const float f = rows.scale(a, big, own) * (a.scale * kLog2e);
        st.run(rows, w.lo, kStep, f, sc);
        keep_part<BITS, D, NT>(k, slot, w, a, 0, lane, rows);
    });
}

// A tile of one of the workgroups that have many rows, for many_rows(), which has two steps on their way where
// the registers suffice: 40 x 2 to 5 tokens of 16 heads of 64 behind four prefixes, 4 bits, 104 us with one,
// 83 with two and three workgroups a CU in the place of two; leaving out the steps of waves without rows 80.
struct Piece {
    const Share& w;
    const Kept& k;
    int64_t slot;
    template <int BITS, int D, int NC>
    __device__ void keep(const Share& s, const KvAttend& a, int r0, int lane,
                         const Rows<BITS, D, NC>& r) const {
        keep_part<BITS, D, NC>(k, slot, s, a, r0, lane, r);
    }
};
template <int BITS, int D, int NC, int W>
constexpr int ahead_of<Piece, BITS, D, NC, W> = D == 256 && W == 8 ? 1 : 2;  // registers
template <class B>
__device__ inline Share share_of(const KvCache&, const B&, const KvAttend&, const Plan&, const Piece& x) {
    return x.w;
}

// How a launch's workgroups are dealt out: to the prefixes and to what stands behind, so that both end
// together.  The cost of a step of each is that of a workgroup (of four waves' steps behind).
struct Deal {
    int places;
    float lead, own;
};

__device__ inline int dealt(const Deal& d, int lead, int own) {
    if (lead == 0 || own == 0) return lead ? d.places : 0;
    const float x = lead * d.lead, y = own * d.own;
    return min(d.places - 1, max(1, static_cast<int>(d.places * x / (x + y) + 0.5f)));
}

// Workgroups of a CU, as the registers allow: heads of 64 in 4 bits 85.0 us with three and 81.5 with four
// (40 x 2 to 5 tokens behind four prefixes), which spill 6 registers; in 8 bits, where four spill more,
// 39.4 and 46.9 (4 behind 50000).  Two of heads of 128 in 8 bits spill one.
constexpr int both_waves(int bits, int D) { return D == 256 ? 1 : D == 128 ? 2 : bits == 4 ? 4 : 3; }

// Prefixes and what stands behind them in one launch, so that the former, many rows, which vector and matrix
// instructions bound, run beside the latter, which reading the cache bounds: 64 tokens of 32 heads on 8 of
// 128 behind 16003, 50 to 1500 of their own, 8 bits: 66.5 us a call, join included, and 80 in two launches
// (64 now; in a trace, one by one, 62 and 10 the join).  Of it 2.5 us go by before the first load of codes, 8 to write the parts; a step of 128 rows takes 3.0 us
// with two such workgroups on a CU and 3.3 to 3.8 beside waves that read (VALU 40% of the cycles, matrix
// cores 17%, waves wait in 49% of theirs).  LEAD: 0 few rows before, else tiles of 64 LEAD.  Tiles of 128
// rows are turned to float16 half as often, but leave less beside them; us: the case above 64.2 a call and
// 69.5 with tiles of 64, of heads of 64 48.8 and 44.6, 64 tokens of 16 heads on 4 of 256 96 and 88, 48 behind
// three prefixes 62.3 and 51.5.
constexpr int most_lead(int D) { return D == 128 ? 2 : 1; }

template <int BITS, int D, int LEAD>
__global__ __launch_bounds__(256, (both_waves(BITS, D)))
void kv_both_kernel(KvCache c, KvOwn b, KvLead lead, KvAttend a, KvAttend la, Kept ok, Kept lk, Deal d) {
    __shared__ __align__(16) float few[4][192];
    const int lane = threadIdx.x & 63, wave = wave_id(), block = blockIdx.x;
    const int lt = all_steps(c, lead, lane, [&](const KvSeq& s) { return tile_steps(lead, s, la, lk); }).sum;
    const int ot = all_steps(c, b, lane, [&](const KvSeq& s) { return tile_steps(b, s, a, ok); }).sum;
    const int n = dealt(d, lt, ot);
    if (block >= n) {
        few_steps<BITS, D, 1>(c, b, a, ok, ot, (d.places - n) * 4, (block - n) * 4 + wave, lane, few[wave]);
        return;
    }
    if constexpr (LEAD == 0) {
        few_steps<BITS, D, 1>(c, lead, la, lk, lt, n * 4, block * 4 + wave, lane, few[wave]);
    } else {
        JHQ_MANY_LDS(BITS, D, 4);
        each_tile(c, lead, la, lk, lt, n, 1, block, lane, threadIdx.x == 0, [&](const Share& w, int64_t slot) {
            many_rows<BITS, D, LEAD, 4>(c, lead, la, Plan{}, Piece{w, lk, slot}, kf, vf, sc, bigs);
        });
    }
}

// More rows behind the prefixes too: tiles of 16 NC W rows on both sides.
template <int BITS, int D, int NC, int W>
__global__ __launch_bounds__(64 * W, W == 8 || D < 256 ? 2 : 1)
void kv_tiles_kernel(KvCache c, KvOwn b, KvLead lead, KvAttend a, KvAttend la, Kept ok, Kept lk, Deal d) {
    JHQ_MANY_LDS(BITS, D, W);
    const int lane = threadIdx.x & 63, block = blockIdx.x;
    const int lt = all_steps(c, lead, lane, [&](const KvSeq& s) { return tile_steps(lead, s, la, lk); }).sum;
    const int ot = all_steps(c, b, lane, [&](const KvSeq& s) { return tile_steps(b, s, a, ok); }).sum;
    const int n = dealt(d, lt, ot);
    if (block < n)
        each_tile(c, lead, la, lk, lt, n, 1, block, lane, threadIdx.x == 0, [&](const Share& w, int64_t slot) {
            many_rows<BITS, D, NC, W>(c, lead, la, Plan{}, Piece{w, lk, slot}, kf, vf, sc, bigs);
        });
    else
        each_tile(c, b, a, ok, ot, d.places - n, 1, block - n, lane, threadIdx.x == 0,
                  [&](const Share& w, int64_t slot) {
                      many_rows<BITS, D, NC, W>(c, b, a, Plan{}, Piece{w, ok, slot}, kf, vf, sc, bigs);
                  });
}

// The parts of a row: their number, the first one's place and the way to the others, sums of values
// and (maximum, sum).
struct Parts {
    int n;
    int64_t first, next, jump;
    const float *o, *ml;
    __device__ int64_t at(int k) const { return first + k * next + (k ? jump : 0); }
};

// Of row x (token i, query head h) of sequence seq.
__device__ inline Parts parts_of(const Kept& k, const KvSeq& s, int seq, int i, int h, int H, const KvAttend& a,
                                 int D) {
    const int x = i * a.G + h % a.G;
    const int2 j = k.joins[(first_tile(k, s, seq, a.G) + x / k.tile) * H + h / a.G];
    // one worker has had it all
    if (j.y == 0) return {1, (s.row + i) * a.heads + h, 0, 0, k.whole, k.whole + k.rows * D};
    return {j.y + 1, static_cast<int64_t>(2 * j.x + 1) * k.tile + x % k.tile, 2 * static_cast<int64_t>(k.tile),
            -static_cast<int64_t>(k.tile), k.slots, k.slots + k.n * k.tile * D};
}

// Joins what the passes have of a row; latency and reading the parts bound it.  A thread has 4
// elements of every Y-th part: 2048 rows of 20 parts of 128 elements 9.9 us with 4 (9.7 now), 10.2 with 2, 10.9
// with 1, 13.5 with 8.  Fewer rows have more parts each, and a workgroup of its own each; calls with workgroups of
// several rows, of one, of one with 512 threads, us (32 heads on 8 of 128, 8 bits): 32 tokens behind 16000
// (1024 rows) 43.0, 42.4, 46.5; 16 33.2, 31.9, 32.7; 4 behind 50000 45.4, 41.6, 40.4, on heads of 64 36.8,
// 28.6, 27.9; 4 of 8 heads on 2 behind 100000 56.7, 41.1, 34.7.
constexpr int kJoinWays = 4;
constexpr int64_t join_rows(int D) { return 256 / (D / 4 * kJoinWays); }  // of a workgroup

template <int D, int Y, int N>
__global__ __launch_bounds__(N) void kv_shared_join_kernel(KvCache c, KvOwn b, KvLead lead, KvAttend a,
                                                             Kept lk, Kept ok) {
    constexpr int T = D / 4, R = N / (T * Y);
    static_assert(Y > 1 && T * Y % 64 == 0, "a wave's threads have one row");
    __shared__ __align__(16) float acc[R][Y][D];
    __shared__ float ml[R][Y][2];
    const int t = threadIdx.x % T, y = threadIdx.x / T % Y, r = threadIdx.x / (Y * T);
    const int x = blockIdx.x * R + __builtin_amdgcn_readfirstlane(r);
    const int tok = x / a.heads, h = x - tok * a.heads;
    const int seq = last_at_most(b.n_seq, tok, [&](int j) { return b.cu_q[j]; });
    const int grp = last_at_most(lead.n_seq, tok, [&](int j) { return lead.cu_q[j]; });
    const KvSeq s = kv_seq(b, seq, c.shift);
    const int64_t i = tok - s.row;
    const bool has = x < lk.rows && i >= 0 && i < s.q;
    bool good = s.ok, sees = false;
    Parts A = {}, O = {};
    if (has && good) {
        sees = sees_any(s, a, static_cast<int>(i));
        O = parts_of(ok, s, seq, static_cast<int>(i), h, c.H, a, D);
        const KvSeq w = kv_seq(lead, grp, c.shift);
        const int64_t li = tok - w.row;
        // What the sequence leaves out in front has to be what its row's group has read: a group with a prefix
        // has whole sequences, not the end of one that begins before it.
        if (tok >= lead.cu_q[grp] && tok < lead.cu_q[grp + 1])
            good = w.ok && li < w.q && s.from == w.n &&
                   (w.n == 0 || (s.row >= w.row && s.row + s.q <= w.row + w.q));
        else
            good = s.from == 0;
        if (good && s.from) {
            sees = true;
            A = parts_of(lk, w, grp, static_cast<int>(li), h, c.H, a, D);
        }
    }
    float m = kNone, l = 0.0f;
    f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int k = y; k < A.n + O.n; k += Y) {
        const bool own = k >= A.n;
        const int64_t at = own ? O.at(k - A.n) : A.at(k);
        const float2 st = *reinterpret_cast<const float2*>((own ? O.ml : A.ml) + at * 2);
        const f4 v = *reinterpret_cast<const f4*>((own ? O.o : A.o) + at * D + t * 4);
        const float big = fmaxf(m, st.x);
        const float f0 = __builtin_amdgcn_exp2f(m - big), f1 = __builtin_amdgcn_exp2f(st.x - big);
        l = fmaf(l, f0, st.y * f1);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(o[e], f0, v[e] * f1);
        m = big;
    }
    *reinterpret_cast<f4*>(acc[r][y] + t * 4) = o;
    if (t == 0) {
        ml[r][y][0] = m;
        ml[r][y][1] = l;
    }
    __syncthreads();
    if (y) return;
    l = 0.0f;
    o = f4{0, 0, 0, 0};
#pragma unroll
    for (int z = 0; z < Y; z++) m = fmaxf(m, ml[r][z][0]);
#pragma unroll
    for (int z = 0; z < Y; z++) {
        const float f = __builtin_amdgcn_exp2f(ml[r][z][0] - m);
        l = fmaf(ml[r][z][1], f, l);
        o += *reinterpret_cast<const f4*>(acc[r][z] + t * 4) * f;
    }
    if (!has) return;
    const int64_t row = static_cast<int64_t>(tok) * a.heads + h;
    const float bad = nan32();
    store4(a, row * D + t * 4, good ? o * inverse_of(l, sees) : f4{bad, bad, bad, bad});
    if (a.lse && t == 0) a.lse[row] = good ? lse_of(m, l, sees) : bad;
}

// What a call runs.
struct Both {
    bool shared;    // false: attention as without a prefix
    bool few;       // 16 rows at most behind the prefix
    int lead;       // column tiles of a wave over the prefix, 0: few rows there too
    int waves;      // of a workgroup
    int places;     // workgroups of the launch
    Kept lk, ok;
    int64_t work;   // bytes, -1: more than 2^50 (of attention as without a prefix)
};

// Whether a prefix is read once, by estimates of both ways from the call's bounds (the longest prefix
// stands for all): reading the cache at 5 TB/s or, over more rows than a wave takes for itself, steps
// of tiles, whichever is longer; and for the passes' parts 5.5 us, 150 ns a sequence and, at 128
// elements, 1.7 ns a row.  Measured, attention of every sequence and with the prefix read once, us (32
// heads on 8 of 128, 8 bits, up to 200 tokens of their own): single tokens, 64 behind 900 28.6 and
// 28.4, behind 4000 65.5 and 37.0; 8 behind 2000 19.4 and 20.8, behind 4000 23.5 and 21.6, behind
// 16000 48.6 and 30.0; 3 behind 4000 16.5 and 19.1, behind 8000 21.3 and 19.9; chunks of up to 16, 12
// behind 2000 31.5 and 43.6, behind 8000 89.6 and 68.2; of up to 80, 32 behind 8000 543 and 501,
// behind 2000 178 and 256.
bool worth(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G) {
    const double step = (D == 64 ? 3.0 : D == 128 ? 5.0 : 15.0) * c.H * (lead.max_kv / kStep + 1);  // ns
    const double read = (2.0 * (c.codes >> c.shift) + 8) * c.H * lead.max_kv / 5000;
    const double rows = static_cast<double>(b.max_q) * G, before = static_cast<double>(lead.max_q) * G;
    const double all = static_cast<double>(b.n_tokens) * G;
    auto tiles = [&](double each, int n, double most) {
        return each <= few_rows(D) ? 0.0 : std::min(n * std::ceil(each / most), all / most + n);
    };
    // sequences without new tokens cost nothing
    const int n = static_cast<int>(std::min<int64_t>(b.n_seq, b.n_tokens));
    const int groups = static_cast<int>(std::min<int64_t>(lead.n_seq, b.n_tokens));
    const double every = std::max(n * read, tiles(rows, n, rows <= 64 ? 64 : 128) * step);
    const double once = std::max(groups * read, tiles(before, groups, before <= 64 ? 64 : 128) * step);
    return every > once + 5500 + 150.0 * n + 1.7 * D / 128 * all * c.H;
}

Both choose_both(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G, bool once, float* work) {
    Both r = {};
    const int64_t rows = static_cast<int64_t>(b.max_q) * G, before = static_cast<int64_t>(lead.max_q) * G;
    const int64_t all = b.n_tokens * c.H * G;
    r.few = rows <= 16;
    const int64_t longest = std::max(rows, before);
    r.lead = longest <= 16 ? 0 : longest <= 64 ? 1 : r.few ? most_lead(D) : 2;
    r.waves = D == 256 && r.lead == 2 ? 8 : 4;
    const int bits = (c.codes >> c.shift) * 8 / D;
    r.places = 256 * (r.few ? both_waves(bits, D) : D == 256 ? 1 : 2);
    const int tile = r.lead ? 64 * r.lead : 16, own = r.few ? 16 : tile;
    if (r.waves == 8) r.lead = 1;
    // Numbers of tiles, of which first_tile leaves as many; steps are numbered with an int, also where
    // cu_q does not ascend and every sequence has as many rows as the bounds allow.
    const int64_t tiles = b.n_tokens * G / tile + lead.n_seq, own_tiles = b.n_tokens * G / own + b.n_seq;
    const __int128 steps = (static_cast<__int128>(lead.n_seq) * (before / tile + 1) * (lead.max_kv / kStep + 8) +
                            static_cast<__int128>(b.n_seq) * (rows / own + 1) * (b.max_kv / kStep + 8)) * c.H;
    // and the join is one launch: all below 2^31 / D
    r.shared = lead.n_seq > 0 && lead.max_kv > 0 && steps < INT32_MAX / 2 && all < join_rows(D) << 23 &&
               (once || worth(c, lead, b, D, G));
    if (!r.shared) {
        r.work = kv_attend_work(c, b, D, G, 0);
        return r;
    }
    const int64_t floats = lay_out(r.lk, work, D, 2 * r.places * (r.lead ? 1 : 4), tile, tiles * c.H, all);
    r.work = (floats + lay_out(r.ok, work + floats, D, 2 * r.places * (r.few ? 4 : 1), own, own_tiles * c.H, all)) * 4;
    r.lk.start = 3;
    r.ok.start = r.few ? 1 : 3;
    return r;
}

template <int BITS, int D>
hipError_t launch(const KvCache& c, const KvBatch& lead, const KvBatch& b, const KvAttend& a,
                  const Both& ch, hipStream_t s) {
    KvLead lb;
    static_cast<KvBatch&>(lb) = lead;
    KvOwn ob;
    static_cast<KvBatch&>(ob) = b;
    ob.lead_cu = lead.cu_q;
    ob.lead_len = lead.kv_len;
    ob.n_lead = lead.n_seq;
    KvAttend la = a;
    la.causal = 0;
    // measured: 64 single tokens behind 16003, 8 bits, 32 heads on 8 of 128: 67.1 us with 0.22, 64.6 with 0.3,
    // 65.6 with 0.4, 67.1 with 0.5, 71.3 with 0.65; of 64 56.6 with 0.2, 48.4 with 0.3, 45.9 with 0.4, 44.7
    // with 0.5; 16 on 4 of 256, three prefixes, 59.6, 51.7, 52.9, 53.2
    const float own = D == 64 || ch.lead == 1 && D == 128 ? 0.4f : 0.3f;
    const Deal d = {ch.places, 1.0f, ch.few && ch.lead ? own : 1.0f};
    auto go = [&](auto kernel) {
        kernel<<<ch.places, 64 * ch.waves, 0, s>>>(c, ob, lb, a, la, ch.ok, ch.lk, d);
    };
    if (ch.few && ch.lead == 0)
        go(kv_both_kernel<BITS, D, 0>);
    else if (ch.few && ch.lead == 1)
        go(kv_both_kernel<BITS, D, 1>);
    else if (ch.few)
        go(kv_both_kernel<BITS, D, most_lead(D)>);
    else if (ch.lead == 1 && ch.waves == 4)
        go(kv_tiles_kernel<BITS, D, 1, 4>);
    else if constexpr (D == 256)
        go(kv_tiles_kernel<BITS, D, 1, 8>);
    else
        go(kv_tiles_kernel<BITS, D, 2, 4>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t rows = ch.lk.rows;
    auto join = [&](auto kernel, int64_t blocks, int threads) {
        kernel<<<static_cast<unsigned>(blocks), threads, 0, s>>>(c, ob, lb, a, ch.lk, ch.ok);
    };
    if (rows <= 128)
        join(kv_shared_join_kernel<D, 2048 / D, 512>, rows, 512);
    else if (rows <= 1024)
        join(kv_shared_join_kernel<D, 1024 / D, 256>, rows, 256);
    else
        join(kv_shared_join_kernel<D, kJoinWays, 256>, (rows + join_rows(D) - 1) / join_rows(D), 256);
    return hipGetLastError();
}

}  // namespace

int64_t kv_shared_work(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G, bool once) {
    return choose_both(c, lead, b, D, G, once, nullptr).work;
}

hipError_t kv_attend_shared(const KvCache& c, const KvBatch& lead, const KvBatch& b, int bits, int D,
                            const KvAttend& a, bool once, hipStream_t s) {
    const Both p = choose_both(c, lead, b, D, a.G, once, a.work);
    if (!p.shared) return kv_attend(c, b, bits, D, a, s);
    if (bits == 8)
        return D == 64    ? launch<8, 64>(c, lead, b, a, p, s)
               : D == 128 ? launch<8, 128>(c, lead, b, a, p, s)
                          : launch<8, 256>(c, lead, b, a, p, s);
    return D == 64    ? launch<4, 64>(c, lead, b, a, p, s)
           : D == 128 ? launch<4, 128>(c, lead, b, a, p, s)
                      : launch<4, 256>(c, lead, b, a, p, s);
}

}  // namespace jhq
