// kv_attend.h — attention of new tokens over the quantised key/value cache: its arithmetic and its
// kernels.  Internal to kv_attend.hip and kv_shared.hip.
//
// Mathematics.  With codes c and scales of the cache, s_ij = scale * ks_j <q_i,
// ck_j> and o_i = sum_j w_ij vs_j cv_j / sum_j w_ij, w_ij = exp(s_ij).  Both
// products run on the matrix cores (f32_16x16x32_f16) on the codes themselves:
// a code is exact in float16, queries are exact there too once the largest is
// scaled to 2^14 (only what is 2^-28 of it becomes subnormal; rows much smaller than
// their neighbours have a scale of their own), and sums are float32.  The scales go
// where they cost one operation per score:
//   a_ij  = S_ij * (scale log2e ks_j) + log2 vs_j
//   p'_ij = 2^(a_ij - m_i)            = w_ij vs_j 2^-m_i
//   l_i   = sum_j p'_ij / vs_j          o_i = sum_j p'_ij cv_j / l_i
// m_i is a running maximum of a_ij less 9, so p' is rounded to float16 relative to the
// row's largest weighted scale whatever the sizes of the values, and in the upper part
// of float16's range: the largest p' is 2^9 to 2^15, one of 2^-23 of it still has 11
// bits, and only what is below 2^-34 of it is lost from o_i (of 2^20 tokens 2^-14).  A
// value scale of 0 (all codes 0) counts as 2^-80, below any scale the cache holds.  The price is
// range: p' / vs is lost where p' is below 2^-126, so a weight w_max 2^-24 is in l_i as
// long as scales differ by less than 2^111 (l_i without the scale would take a second
// exponential, and the one is a quarter of the time with many rows).  m_i moves
// only when some a_ij passes the maximum that it stands for by more than 6 (p' <=
// 2^15): then, and not at every step, sums and accumulators are rescaled.
//
// Layout.  Scores are computed transposed, S^T = K Q^T: a lane of the result
// holds one query row (column lane % 16) and 4 tokens, so a row's statistics
// live in its lane.  Tile t of a step of 64 tokens takes as its row 4 g + i the
// token 16 g + 4 t + i.  Then lane group g = lane / 16 ends with the scores of
// the tokens 16 g .. 16 g + 15 of its rows, which is, in order, what it has to
// supply to O^T = V^T P^T, and the 16 bytes [element][16 tokens] of the cache's
// values are what it has to supply of V^T: nothing crosses lanes.
#pragma once
#include "kvcache.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace jhq {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;          // tokens of a step
// Steps of a streaming wave at least: 8 sequences of 2000 tokens 13.7 us with two, 14.9 with
// one, 17.0 with four.
constexpr int kLeast = 2;
// Sequences up to which tiles are numbered by their place from the end, which takes a sum over
// all sequences for every bit of their number: a lane holds one.  Tiles of more are numbered one
// sequence after the other, in one pass.  New tokens over 300 more, 32 heads on 8 of 128: 1024 of 1 to
// 58 791 us sorted and 600 not, 512 of 1 to 117 608 and 491, 128 of 1 to 468 482 and 460; 12 of 64:
// 128 of 234 136, 141; 64 of 468 150, 163.  12 windowed chunks on heads of 256: 115, 160.
constexpr int kSorted = 64;
// Tokens that one workgroup takes alone: one sequence of 1000 tokens 9.7 us so and 11.8
// streaming, of 2000 13.9 and 11.8; 64 of 1000 27.1 and 29.6.
constexpr int kShortSpan = 1024;
constexpr float kNone = -FLT_MAX;  // running maximum before the first token
// log2 of the largest weight where the maximum has just moved, and how far a score may pass
// that maximum before it moves again.  11 and 4 hold weights down to 2^-36 and move it more
// often (the 4-bit passages of 64-wide heads 86.8 us with 0 and 8, 87.3 with 9 and 6, 87.8 with
// 11 and 4).
constexpr float kHead = 9.0f, kSlack = 6.0f;
constexpr float kHeadPart = 0x1p-9f;  // 2^-kHead
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Whether a batch's rows see only a part of their tokens in a pass.
template <class B>
constexpr bool kParts = !std::is_same<B, KvBatch>::value;

// The wave's number in its workgroup, as a value the compiler knows to be uniform.
__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ inline float nan32() { return __uint_as_float(0x7fc00000u); }

// Sizes that follow from the cache's bits and the head's elements.
template <int BITS, int D>
struct Dim {
    static constexpr int ROW = D * BITS / 8;        // bytes of a row
    static constexpr int LB = ROW / 4;              // of them in a lane's key operand
    static constexpr int NU = LB < 16 ? 1 : LB / 16;  // loads that bring them
    static constexpr int KS = D / 32;               // products along D
    static constexpr int ET = ROW / 16;             // tiles of value byte columns
    static constexpr int DT = D / 16;               // tiles of output elements
    // First byte column of octet o (8 bytes) of lane group g.
    __device__ static int octet(int o, int g) {
        return LB == 8 ? g * 8 : ((o >> 1) * 4 + g) * 16 + (o & 1) * 8;
    }
};

template <int LB>
struct KeyReg {
    typedef u4 type;
};
template <>
struct KeyReg<8> {
    typedef u2 type;
};

// 8 bytes of 8-bit codes as float16: 0x6400 | u is 1024 + u.
__device__ inline h8 half8(uint32_t a, uint32_t b) {
    const h2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const uint32_t k = 0x64646464u;
    h2 r[4] = {__builtin_bit_cast(h2, __builtin_amdgcn_perm(a, k, 0x00050004)) + bias,
               __builtin_bit_cast(h2, __builtin_amdgcn_perm(a, k, 0x00070006)) + bias,
               __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, k, 0x00050004)) + bias,
               __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, k, 0x00070006)) + bias};
    return __builtin_bit_cast(h8, r);
}

// 8 bytes of 4-bit codes: low and high nibbles, in the byte order 0 2 1 3 4 6 5 7.
__device__ inline void half4(uint32_t a, uint32_t b, h8& lo, h8& hi) {
    const h2 lob = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
    const h2 hib = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
    const h2 sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const uint32_t w[4] = {a, a >> 8, b, b >> 8};
    // 1024 twice, in a register: with two constants in it, "and, or" is not one
    // instruction
    uint32_t k = 0x64006400u;
    asm("" : "+v"(k));
    h2 l[4], h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        l[i] = __builtin_bit_cast(h2, (w[i] & 0x000f000fu) | k) + lob;
        // 1024 + 16 n
        h[i] = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w[i] & 0x00f000f0u) | k), sixteenth,
                                         hib);
    }
    lo = __builtin_bit_cast(h8, l);
    hi = __builtin_bit_cast(h8, h);
}

// Place of operand element i of an octet within it.
template <int BITS>
__device__ constexpr int place(int i) {
    return BITS == 8 ? i : (i & 4) | ((i & 1) << 1) | ((i >> 1) & 1);
}

__device__ inline f4 mfma(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ inline float value16(const KvAttend& a, uint32_t h) {
    return a.dtype == JHQ_BF16
               ? __uint_as_float(h << 16)
               : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}

// How the work is cut; made on the host by choose().
struct Plan {
    int tile;     // rows of a tile
    int tiles;    // tiles of a sequence with max_q new tokens
    int64_t real; // tiles of all sequences at most
    int log_workers;  // of the streaming kernel, a power of two
    int nsplit;   // parts that a tile's tokens may be cut into (many rows)
    int chunk;    // tokens of a part, a multiple of kStep
    int64_t rows; // of the partial results: n_tokens * query heads
    int per;      // tokens that the join takes for a sequence, 0: it goes over rows
};

// Rows of one head of one sequence, and tokens that they attend to.
struct Share {
    KvSeq s;
    int seq, head, split;
    int r0, rn;      // rows of the sequence: token i of head h*G+g is row i*G+g
    int lo, hi;      // tokens [lo, hi), lo a multiple of kStep
    int full_lo, full_hi;  // tokens that every row sees
    bool any;
    bool alone;      // no other part of these rows
};

// Positions seen by new token i: [first, last).
__device__ inline int see_hi(const KvSeq& s, const KvAttend& a, int i) {
    return a.causal ? max(0, min(s.n - s.q + i + 1, s.n)) : s.n;
}
__device__ inline int see_lo(const KvSeq& s, const KvAttend& a, int i) {
    return max(a.window ? max(0, s.n - s.q + i + 1 - a.window) : 0, s.from);
}
__device__ inline bool sees_any(const KvSeq& s, const KvAttend& a, int i) {
    return see_hi(s, a, i) > see_lo(s, a, i);
}

// The tokens that rows [r0, r0 + rn) of a share's sequence attend to.
__device__ inline void span_of(Share& r, const KvAttend& a) {
    const int i0 = r.r0 / a.G, i1 = (r.r0 + r.rn - 1) / a.G;
    r.lo = see_lo(r.s, a, i0) / kStep * kStep;
    r.hi = see_hi(r.s, a, i1);
    r.full_lo = see_lo(r.s, a, i1);
    r.full_hi = see_hi(r.s, a, i0);
}

// The sum over a full wave, uniform: along rows of 16 lanes, then from row to row.
__device__ inline int wave_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return __builtin_amdgcn_readlane(x, 63);
}

// The lane's sequence of 64, no new token past the last.
template <class B>
__device__ inline KvSeq lane_seq(const KvCache& c, const B& b, int s) {
    if (s < b.n_seq) return kv_seq(b, s, c.shift);
    return {0, 0, 0, true, 0};
}

// Tiles of sequence s, none past the last.
__device__ inline int tiles_of(const KvCache& c, const KvBatch& b, const KvAttend& a, const Plan& p,
                               int s) {
    return (lane_seq(c, b, s).q * a.G + p.tile - 1) / p.tile;
}

// The i-th tile of those that the sequences have, one sequence after the other; false past the
// last.
__device__ inline bool tile_in_order(const KvCache& c, const KvBatch& b, const KvAttend& a,
                                     const Plan& p, int i, int* seq, int* tile) {
    const int lane = threadIdx.x & 63;
    for (int x = 0; x < b.n_seq; x += 256) {
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; u++) n[u] = tiles_of(c, b, a, p, x + u * 64 + lane);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int sum = wave_sum(n[u]);
            if (i < sum) {
                int in = n[u];  // inclusive sum
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int y = __shfl_up(in, o);
                    if (lane >= o) in += y;
                }
                const int k = __builtin_ctzll(__ballot(in > i));
                *seq = x + u * 64 + k;
                *tile = i - __builtin_amdgcn_readlane(in - n[u], k);
                return true;
            }
            i -= sum;
        }
    }
    return false;
}

// The i-th tile of those that the sequences have, in the order of their numbers from each
// sequence's end, then of the sequences; false past the last.  Tile numbers below t have
// sum_s min(tiles_s, t) tiles, which is searched for i.
__device__ inline bool tile_at(const KvCache& c, const KvBatch& b, const KvAttend& a, const Plan& p,
                               int i, int* seq, int* tile) {
    const int lane = threadIdx.x & 63;
    const int first = tiles_of(c, b, a, p, lane);
    auto below = [&](int t) {
        int n = min(first, t);
        for (int s = lane + 64; s < b.n_seq; s += 64) n += min(tiles_of(c, b, a, p, s), t);
        return wave_sum(n);
    };
    if (i >= below(p.tiles)) return false;
    int lo = 0, hi = p.tiles - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (below(mid) <= i)
            lo = mid;
        else
            hi = mid - 1;
    }
    int r = i - below(lo);
    for (int x = 0; x < b.n_seq; x += 64) {
        const uint64_t has = __ballot((x ? tiles_of(c, b, a, p, x + lane) : first) > lo);
        const int n = __builtin_popcountll(has);
        if (r < n) {
            const int before = __builtin_amdgcn_mbcnt_hi(
                static_cast<uint32_t>(has >> 32),
                __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(has), 0));
            *seq = x + __builtin_ctzll(__ballot((has >> lane & 1) && before == r));
            *tile = lo;
            return true;
        }
        r -= n;
    }
    return false;
}

// A workgroup's tile of rows and part of their tokens.
__device__ inline Share share_of(const KvCache& c, const KvBatch& b, const KvAttend& a,
                                 const Plan& p, uint32_t block) {
    Share r;
    // Heads vary fastest (workgroups go round the 8 XCDs, whose L2 caches then
    // hold few heads each), then sequences, then tiles from the last, which sees
    // most (of many sequences: sequence by sequence), then parts.  Of several only the tiles
    // that they have are counted, so that the XCDs get equally many whatever the lengths.
    // 12 chunks of 1 to 1500 tokens, window 1024, 8 heads on 4 of 256: 118 us, and 163
    // counting as many for each sequence, where two heads' sequences of one parity shared an
    // XCD; 10 of 100 to 700, 12 heads of 64, whose keys then lay in one XCD's L2: 87 and 84.
    const uint32_t w = block / c.H, real = static_cast<uint32_t>(p.real);
    r.head = block % c.H;
    r.split = w / real;
    int tile = w % real;
    r.seq = 0;
    r.any = false;
    if (p.tiles == 1) {
        r.seq = tile;
        tile = 0;
    } else if (b.n_seq > kSorted) {
        if (!tile_in_order(c, b, a, p, tile, &r.seq, &tile)) return r;
    } else if (b.n_seq > 1 && !tile_at(c, b, a, p, tile, &r.seq, &tile)) {
        return r;
    }
    r.s = kv_seq(b, r.seq, c.shift);
    const int rows = r.s.q * a.G, mine = (rows + p.tile - 1) / p.tile - 1 - tile;
    r.r0 = mine * p.tile;
    r.rn = min(p.tile, rows - r.r0);
    r.any = mine >= 0;
    if (!r.any) return r;
    span_of(r, a);
    r.alone = p.nsplit == 1 || r.hi - r.lo <= p.chunk;
    r.lo += r.split * p.chunk;
    if (p.nsplit > 1) r.hi = min(r.hi, r.lo + p.chunk);
    return r;
}

// Where row r of a share lies: first element of its query, and its output row.
__device__ inline int64_t row_of(const Share& w, const KvAttend& a, int r, int64_t* q) {
    const int i = r / a.G, h = w.head * a.G + (r - i * a.G);
    const int64_t t = w.s.row + i;
    *q = t * a.q.tok + h * a.q.head;
    return t * a.heads + h;
}

// A wave's rows: queries as the second operand of S^T, statistics, sums.
template <int BITS, int D, int NC>
struct Rows {
    using M = Dim<BITS, D>;
    h8 q[NC][M::KS];
    f4 o[NC][M::DT];
    float m[NC], l[NC];
    int hi[NC], lo[NC];  // the row's tokens
    float part[NC];      // what the row's scores are multiplied by where rows are uneven
    bool uneven;         // some part of the wave's is not 1

    // Row 16 k + lane % 16 of the wave's, which start at r0 (the share's last row
    // stands in for rows past it).
    __device__ static int row_at(const Share& w, int r0, int k, int lane) {
        return min(r0 + k * 16 + (lane & 15), w.r0 + w.rn - 1);
    }

    // Sets up the wave's rows and reads their queries as they are.
    __device__ void start(const Share& w, const KvAttend& a, int r0, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int r = row_at(w, r0, k, lane);
            int64_t at;
            row_of(w, a, r, &at);
            hi[k] = see_hi(w.s, a, r / a.G);
            lo[k] = see_lo(w.s, a, r / a.G);
            m[k] = kNone;
            l[k] = 0.0f;
#pragma unroll
            for (int t = 0; t < M::DT; t++) o[k][t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < M::KS; s++) {
                const int64_t e =
                    at + (BITS == 8 ? M::octet(s, g) : M::octet(s >> 1, g) + (s & 1) * (D / 2));
                const uint16_t* const src = static_cast<const uint16_t*>(a.q.p) + e;
                u4 v;
                if (a.q16) {
                    v = *reinterpret_cast<const u4*>(src);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = src[2 * i] | static_cast<uint32_t>(src[2 * i + 1]) << 16;
                }
                q[k][s] = __builtin_bit_cast(h8, v);
            }
        }
    }

    __device__ static float element(const KvAttend& a, u4 v, int i) {
        return value16(a, v[i >> 1] >> (16 * (i & 1)) & 0xffff);
    }

    // The largest finite magnitude of each row's query elements (own, by the lane), and
    // of the wave's: magnitudes of either type are in the order of their bits.
    __device__ float largest(const KvAttend& a, float (&own)[NC]) const {
        const uint32_t inf = a.dtype == JHQ_BF16 ? 0x7f80 : 0x7c00;
        int big = 0;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            us2 two = {0, 0};
#pragma unroll
            for (int s = 0; s < M::KS; s++) {
                const u4 v = __builtin_bit_cast(u4, q[k][s]);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    two = __builtin_elementwise_max(two, __builtin_bit_cast(us2, v[i] & 0x7fff7fffu));
            }
            uint32_t row = max(two[0], two[1]);
            if (__any(row >= inf)) {
                row = 0;
#pragma unroll
                for (int s = 0; s < M::KS; s++) {
                    const u4 v = __builtin_bit_cast(u4, q[k][s]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t x = v[i] & 0x7fff, y = v[i] >> 16 & 0x7fff;
                        row = max(row, max(x < inf ? x : 0, y < inf ? y : 0));
                    }
                }
            }
            int r = static_cast<int>(row);
            r = max(r, __shfl_xor(r, 16));
            r = max(r, __shfl_xor(r, 32));
            own[k] = value16(a, r);
            big = max(big, r);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) big = max(big, __shfl_xor(big, o));
        return value16(a, big);
    }

    // The power of two that takes x to 2^13 .. 2^14.
    __device__ static int exponent(float x) {
        int e = 0;
        if (x > 0.0f) {
            frexpf(x, &e);
            e = max(-126, min(126, 14 - e));
        }
        return e;
    }

    // Turns the queries to operands, scaled by the power of two that takes big, the
    // largest of the workgroup's, to 2^13 .. 2^14; returns its inverse, which S has to be
    // multiplied by.  A row that is smaller than big by more than 2^-16, of which that
    // would leave too little, is scaled by its own, and its scores by the quotient.
    __device__ float scale(const KvAttend& a, float big, const float (&own)[NC]) {
        const int e = exponent(big);
        bool any = false;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int ek = own[k] > 0.0f && own[k] < big * 0x1p-16f ? exponent(own[k]) : e;
            any |= ek != e;
            part[k] = ldexpf(1.0f, e - ek);
            const float f = ldexpf(1.0f, ek);
#pragma unroll
            for (int s = 0; s < M::KS; s++) {
                const u4 v = __builtin_bit_cast(u4, q[k][s]);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    q[k][s][i] = static_cast<_Float16>(element(a, v, place<BITS>(i)) * f);
            }
        }
        uneven = __any(any);
        return ldexpf(1.0f, -e);
    }

    // Scores of half a step (its tiles 2 hf, 2 hf + 1) to weights.  s[k][t][i]: token
    // j0 + 16 g + 8 hf + 4 t + i.  sc: the step's kk, lv and iv (64 floats each).
    __device__ void weigh(f4 (&s)[NC][2], const float* sc, int lane, int j0, int hf, bool masked,
                          bool uneven, h8 (&p)[NC]) {
        const int at = (lane >> 4) * 16 + hf * 8;
        const f4* const kk = reinterpret_cast<const f4*>(sc + at);
        const f4* const lv = reinterpret_cast<const f4*>(sc + 64 + at);
        const f4* const iv = reinterpret_cast<const f4*>(sc + 128 + at);
        if (uneven) {
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int t = 0; t < 2; t++) s[k][t] *= part[k];
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const f4 x = kk[t], y = lv[t];
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[k][t][i] = fmaf(s[k][t][i], x[i], y[i]);
        }
        if (masked) {
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int h = hi[k] - j0 - at, l0 = lo[k] - j0 - at;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (t * 4 + i >= h || t * 4 + i < l0) s[k][t][i] = -INFINITY;
            }
        }
        float top[NC];
        bool over = false;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            top[k] = s[k][0][0];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top[k] = fmaxf(top[k], s[k][t][i]);
            over |= top[k] > m[k] + (kHead + kSlack);
        }
        if (__any(over)) {
#pragma unroll
            for (int k = 0; k < NC; k++) {
                float n = fmaxf(m[k], top[k] - kHead);
                n = fmaxf(n, __shfl_xor(n, 16));
                n = fmaxf(n, __shfl_xor(n, 32));
                const float f = __builtin_amdgcn_exp2f(m[k] - n);
                m[k] = n;
                l[k] *= f;
#pragma unroll
                for (int t = 0; t < M::DT; t++) o[k][t] *= f;
            }
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const f4 z = iv[t];
#pragma unroll
            for (int k = 0; k < NC; k++) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = __builtin_amdgcn_exp2f(s[k][t][i] - m[k]);
                    l[k] = fmaf(e[i], z[i], l[k]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    p[k][t * 4 + i] = static_cast<_Float16>(e[BITS == 8 ? i : place<4>(i)]);
            }
        }
    }

    // O^T += V^T P^T for half a step and one tile of value byte columns.
    __device__ void add_values(int e, uint32_t w0, uint32_t w1, const h8 (&p)[NC]) {
        if constexpr (BITS == 8) {
            const h8 v = half8(w0, w1);
#pragma unroll
            for (int k = 0; k < NC; k++) o[k][e] = mfma(v, p[k], o[k][e]);
        } else {
            h8 lo8, hi8;
            half4(w0, w1, lo8, hi8);
#pragma unroll
            for (int k = 0; k < NC; k++) {
                o[k][e] = mfma(lo8, p[k], o[k][e]);
                o[k][e + M::ET] = mfma(hi8, p[k], o[k][e + M::ET]);
            }
        }
    }

    // The lanes' sums of a row, joined.
    __device__ void join() {
#pragma unroll
        for (int k = 0; k < NC; k++) {
            l[k] += __shfl_xor(l[k], 16);
            l[k] += __shfl_xor(l[k], 32);
        }
    }
};

// Scores of one tile of 16 tokens.
template <int BITS, int D, int NC>
__device__ inline void score_tile(const typename KeyReg<Dim<BITS, D>::LB>::type (&w)[Dim<BITS, D>::NU],
                                  const Rows<BITS, D, NC>& r, f4 (&s)[NC]) {
    using M = Dim<BITS, D>;
#pragma unroll
    for (int k = 0; k < NC; k++) s[k] = f4{0, 0, 0, 0};
#pragma unroll
    for (int o = 0; o < M::LB / 8; o++) {
        const uint32_t a = w[o >> 1][(o & 1) * 2], b = w[o >> 1][(o & 1) * 2 + 1];
        if constexpr (BITS == 8) {
            const h8 x = half8(a, b);
#pragma unroll
            for (int k = 0; k < NC; k++) s[k] = mfma(x, r.q[k][o], s[k]);
        } else {
            h8 lo, hi;
            half4(a, b, lo, hi);
#pragma unroll
            for (int k = 0; k < NC; k++) {
                s[k] = mfma(lo, r.q[k][2 * o], s[k]);
                s[k] = mfma(hi, r.q[k][2 * o + 1], s[k]);
            }
        }
    }
}

// kk, lv and iv of one token from its scales; dead: past the sequence's end.
__device__ inline void token_terms(float ks, float vs, float f, bool dead, bool lost, float* sc) {
    const bool tiny = vs < 0x1p-80f;  // a NaN is not
    const float kk = ks * f;
    sc[0] = dead ? 0.0f : lost ? nan32() : kk;
    sc[64] = dead ? -INFINITY : tiny ? -80.0f : __builtin_amdgcn_logf(vs);
    // finite also where vs is NaN: a row that does not see the token multiplies it
    // by 0
    sc[128] = dead ? 0.0f : tiny ? 0x1p80f : vs <= FLT_MAX ? __builtin_amdgcn_rcpf(vs) : 0.0f;
}

__device__ inline void store4(const KvAttend& a, int64_t i, f4 x) {
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        h[k] = a.dtype == JHQ_BF16 ? __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[k]))
                                   : __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[k]));
    uint16_t* const p = static_cast<uint16_t*>(a.out) + i;
    if (a.out8) {
        *reinterpret_cast<u2*>(p) = u2{h[0] | h[1] << 16, h[2] | h[3] << 16};
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = static_cast<uint16_t>(h[k]);
    }
}

// What a row's sums of values are multiplied by, and its log-sum-exp.  A sum of 0 is that
// of a row that sees nothing, or of one whose every score is -inf (an infinite query
// element, scores past float32's range): that one's softmax is 0 / 0.
__device__ inline float inverse_of(float l, bool sees) {
    return l == 0.0f ? (sees ? nan32() : 0.0f) : 1.0f / l;
}
__device__ inline float lse_of(float m, float l, bool sees) {
    // both terms without kHead, which would only add to their roundings
    const float x = (m + kHead) + log2f(l * kHeadPart);
    return l == 0.0f ? (sees ? nan32() : -INFINITY) : kLn2 * x;
}

// A share whose sequence is not in order: its rows become NaN.
template <int D>
__device__ void fail_rows(const Share& w, const KvAttend& a, int thread, int threads) {
    const float x = nan32();
    for (int k = thread; k < w.rn * (D / 4); k += threads) {
        int64_t q;
        const int64_t o = row_of(w, a, w.r0 + k / (D / 4), &q);
        store4(a, o * D + k % (D / 4) * 4, f4{x, x, x, x});
        if (a.lse && k % (D / 4) == 0) a.lse[o] = x;
    }
}

// The results of a wave's rows.  Lane group g holds the elements 16 t + 4 g ..
template <int BITS, int D, int NC>
__device__ void finish(const Share& w, const KvAttend& a, int r0, int lane,
                       const Rows<BITS, D, NC>& r) {
    const int g = lane >> 4;
#pragma unroll
    for (int k = 0; k < NC; k++) {
        const int row = r0 + k * 16 + (lane & 15);
        if (row >= w.r0 + w.rn) continue;
        int64_t q;
        const int64_t o = row_of(w, a, row, &q);
        // counted anew: kept through the loop, the row's ends cost 64-wide heads in 4 bits the
        // third wave of a SIMD (86.8 and 94.2 us)
        const bool sees = sees_any(w.s, a, row / a.G);
        const float f = inverse_of(r.l[k], sees);
#pragma unroll
        for (int t = 0; t < D / 16; t++) store4(a, o * D + t * 16 + g * 4, r.o[k][t] * f);
        if (a.lse && g == 0) a.lse[o] = lse_of(r.m[k], r.l[k], sees);
    }
}

// A part of a wave's rows: 16 NC sums per slot, then every slot's maxima and sums.
template <int D, int NC>
__device__ void keep(float* work, int64_t slot, int64_t slots, int rows, int lane, const f4 (&o)[NC][D / 16],
                     const float (&m)[NC], const float (&l)[NC]) {
    const int g = lane >> 4;
#pragma unroll
    for (int k = 0; k < NC; k++) {
        if (k * 16 + (lane & 15) >= rows) continue;
        const int64_t row = slot * (NC * 16) + k * 16 + (lane & 15);
#pragma unroll
        for (int t = 0; t < D / 16; t++)
            *reinterpret_cast<f4*>(work + row * D + t * 16 + g * 4) = o[k][t];
        if (g == 0) {
            float* const ml = work + slots * (NC * 16) * D + row * 2;
            ml[0] = m[k];
            ml[1] = l[k];
        }
    }
}

// Where the bytes of a share's steps lie.  A lane's keys belong to token group
// (lane % 16) / 4 of the step, its values and its token's scales to group lane / 16;
// pages of a step or more are looked up once, for the whole wave.
template <int BITS, int D>
struct Where {
    using M = Dim<BITS, D>;
    const KvCache& c;
    const KvBatch& b;
    const Share& w;
    const int lane;
    int pk, pv;  // pages of the step that look() was last asked for, -1: none

    __device__ Where(const KvCache& c, const KvBatch& b, const Share& w, int lane)
        : c(c), b(b), w(w), lane(lane), pk(-1), pv(-1) {}

    __device__ bool wide() const { return (1 << c.shift) >= kStep; }
    __device__ void look(int j) {
        if (wide()) {
            pk = pv = j < w.s.n ? kv_page(b, c, w.seq, j) : -1;
        } else {
            const int jk = j + (lane >> 2 & 3) * 16, jv = j + (lane >> 4) * 16;
            pk = jk < w.s.n ? kv_page(b, c, w.seq, jk) : -1;
            pv = jv < w.s.n ? kv_page(b, c, w.seq, jv) : -1;
        }
    }
    // Pointers of the step j that was looked up: first key byte of the lane's
    // operand (tile t, load u at + t * 4 ROW + 256 u), first value byte (tile e at +
    // 256 e), scales of the lane's token (keys; values a page on).
    __device__ void find(int j, const uint8_t*& k, const uint8_t*& v, const float*& s) const {
        const int in_page = (1 << c.shift) - 1, at = j & in_page;
        const int g = lane >> 4, kg = lane >> 2 & 3;
        const int klane = (lane & 3) * 16 + (M::LB == 8 ? (g >> 1) * 64 + (g & 1) * 8 : g * 64);
        if (wide()) {
            const uint8_t* const x = kv_block(c, max(__builtin_amdgcn_readfirstlane(pk), 0), w.head);
            k = x + at * M::ROW + (kg * 16 * M::ROW + klane);
            v = x + (c.codes + at * M::ROW) + (g * 16 * M::ROW + (lane & 15) * 16);
            s = reinterpret_cast<const float*>(x + (2 * c.codes + at * 4)) + lane;
        } else {
            const uint8_t* const y = kv_block(c, max(pv, 0), w.head);
            k = kv_block(c, max(pk, 0), w.head) + ((j + kg * 16) & in_page) * M::ROW + klane;
            v = y + c.codes + ((j + g * 16) & in_page) * M::ROW + (lane & 15) * 16;
            s = reinterpret_cast<const float*>(y + 2 * c.codes) + ((j + lane) & in_page);
        }
    }
};

// The cache's bytes of one head as a wave with few rows reads them: keys and
// values go from memory to registers as operands, the next step's loads are
// issued as soon as this step has used the registers.
template <int BITS, int D, int NT>
struct Stream {
    using M = Dim<BITS, D>;
    using K = typename KeyReg<M::LB>::type;
    const KvCache& c;
    const Share& w;
    const int lane;
    Where<BITS, D> where;
    K kr[4][M::NU];
    u4 vr[M::ET];
    float ks, vs;
    bool dead, lost;
    const uint8_t* vp;  // of the step whose keys are loaded

    __device__ Stream(const KvCache& c, const KvBatch& b, const Share& w, int lane)
        : c(c), w(w), lane(lane), where(c, b, w, lane) {}

    __device__ void load_keys(int j) {
        const uint8_t* k;
        const float* s;
        where.find(j, k, vp, s);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int u = 0; u < M::NU; u++)
                kr[t][u] = *reinterpret_cast<const K*>(k + t * (4 * M::ROW) + u * 256);
        ks = s[0];
        vs = s[1 << c.shift];
        dead = j + lane >= w.s.n;
        lost = where.pv < 0;
    }
    __device__ void load_values() {
#pragma unroll
        for (int t = 0; t < M::ET; t++) vr[t] = *reinterpret_cast<const u4*>(vp + t * 256);
    }

    // Issues the first step's loads (at j; nothing where j >= hi).
    __device__ void open(int j, int stride) {
        if (j >= w.hi) return;
        where.look(j);
        load_keys(j);
        load_values();
        if (j + stride < w.hi) where.look(j + stride);
    }

    // The steps j, j + stride, .. below the share's end; sc: 192 floats of LDS, this
    // wave's.
    __device__ void run(Rows<BITS, D, NT>& rows, int j, int stride, float f, float* sc) {
        for (; j < w.hi; j += stride) {
            const int next = j + stride;
            token_terms(ks, vs, f, dead, lost, sc + lane);
            f4 s[2][NT][2];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f4 x[NT];
                score_tile<BITS, D, NT>(kr[t], rows, x);
#pragma unroll
                for (int k = 0; k < NT; k++) s[t >> 1][k][t & 1] = x[k];
            }
            if (next < w.hi) {
                load_keys(next);
                if (next + stride < w.hi) where.look(next + stride);
            }
            // one wave: LDS is written and read in order, the compiler has to keep it
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const bool masked = j < w.full_lo || j + kStep > w.full_hi;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                h8 pr[NT];
                rows.weigh(s[hf], sc, lane, j, hf, masked, rows.uneven, pr);
#pragma unroll
                for (int t = 0; t < M::ET; t++)
                    rows.add_values(t, vr[t][2 * hf], vr[t][2 * hf + 1], pr);
            }
            if (next < w.hi) load_values();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        rows.join();
    }
};

// Few rows (16 NT at most) over short contexts: one workgroup has all tokens of a
// sequence's head, its W waves take every W-th step, and what they have is joined
// in LDS, so that one launch does it.  Latency bounds it (a chain of four loads:
// lengths, page, codes, and the queries beside them): 777 tokens, 2 x 8 rows of
// 128, 9.4 us.  Eight waves, of 256-wide heads four, whose registers would not suffice for more;
// 32 rows of 128 in 8 bits spill seven of them and are faster all the same (64 x 1 over 1000, 2 heads:
// 16.8 us, and 18.3 with four waves).
template <int D>
constexpr int kShortWaves = D == 256 ? 4 : 8;

template <int BITS, int D, int NT, int W>
__global__ __launch_bounds__(64 * W, W / 4) void kv_short_kernel(KvCache c, KvBatch b, KvAttend a,
                                                                 Plan p) {
    using M = Dim<BITS, D>;
    constexpr int R = NT * 16, P = D + 4;
    __shared__ __align__(16) float sc[W][192];
    __shared__ __align__(16) float acc[W][R * P];
    __shared__ float ml[W][R][2];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int g = lane >> 4, r = lane & 15;
    const Share w = share_of(c, b, a, p, blockIdx.x);
    if (!w.any) return;
    if (!w.s.ok) return fail_rows<D>(w, a, threadIdx.x, blockDim.x);
    Rows<BITS, D, NT> rows;
    Stream<BITS, D, NT> st(c, b, w, lane);
    const int j = w.lo + wave * kStep;
    rows.start(w, a, w.r0, lane);
    st.open(j, W * kStep);
    float own[NT];
    const float big = rows.largest(a, own);
    const float f = rows.scale(a, big, own) * (a.scale * kLog2e);
    st.run(rows, j, W * kStep, f, sc[wave]);
#pragma unroll
    for (int k = 0; k < NT; k++) {
#pragma unroll
        for (int t = 0; t < M::DT; t++)
            *reinterpret_cast<f4*>(acc[wave] + (k * 16 + r) * P + t * 16 + g * 4) = rows.o[k][t];
        if (g == 0) {
            ml[wave][k * 16 + r][0] = rows.m[k];
            ml[wave][k * 16 + r][1] = rows.l[k];
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < w.rn * (D / 4); x += 64 * W) {
        const int row = x / (D / 4), e = x % (D / 4) * 4;
        float m = kNone, l = 0.0f;
#pragma unroll
        for (int y = 0; y < W; y++) m = fmaxf(m, ml[y][row][0]);
        f4 o = {0, 0, 0, 0};
#pragma unroll
        for (int y = 0; y < W; y++) {
            const float z = __builtin_amdgcn_exp2f(ml[y][row][0] - m);
            l = fmaf(ml[y][row][1], z, l);
            o += *reinterpret_cast<const f4*>(acc[y] + row * P + e) * z;
        }
        int64_t q;
        const int64_t at = row_of(w, a, w.r0 + row, &q);
        const bool sees = sees_any(w.s, a, (w.r0 + row) / a.G);
        store4(a, at * D + e, o * inverse_of(l, sees));
        if (a.lse && e == 0) a.lse[at] = lse_of(m, l, sees);
    }
}

// Few rows over longer contexts: what bounds it is reading the cache.  The steps
// of all sequences and heads are numbered in one row (sequence, head, step) and
// cut evenly among the waves of the chip, so that ragged batches end together
// whatever their lengths; a wave works alone, from a step within one head to a
// step within another.  What it begins or ends in the middle of a head is kept as
// a part (two at most for a wave: slot 0 where the head began before it, 1 where it
// goes on after it), and kv_join_kernel adds the parts.  The wave that begins a
// head notes which waves have parts of it.
// 64 sequences of 300 to 9000 tokens, 8 heads of 128, 8 bits: 560 MB in 105 us, 5.3 TB/s
// (reading alone reaches 6.2), the parts' sum in 5 more; cut into equal chunks of each
// sequence instead, 149 us.  Four of 130 k tokens, 64 heads on 8 of 128, 4 bits: 425 MB in 83 us, 5.1
// TB/s; there the vector units are busy half of the time.

// Steps of sequence s (a head of it); 0 where it has no new token.
__device__ inline int steps_of(const KvSeq& s, const KvAttend& a, int* lo, int* hi) {
    *lo = see_lo(s, a, 0) / kStep * kStep;
    *hi = see_hi(s, a, s.q - 1);
    // a sequence whose rows see nothing still has rows to write
    return s.q == 0 ? 0 : max(1, (*hi - *lo + kStep - 1) / kStep);
}

// A worker's first step: where it lies, and how many there are.
struct Cut {
    int per, at, end;  // steps of a worker; this one's
    int seq, first;    // the sequence of `at`, and the number of its first step
    KvSeq s;
};

// The steps of all sequences, of which a head of s has steps(s), and what the sum has seen of the lane's
// first sequence, which cut_at begins with.
struct Total {
    int sum, steps;
    KvSeq s;
};

template <class B, class F>
__device__ inline Total all_steps(const KvCache& c, const B& b, int lane, F steps) {
    Total r;
    r.s = lane_seq(c, b, lane);
    r.steps = steps(r.s);
    int sum = r.steps;
    for (int s = lane + 64; s < b.n_seq; s += 64) sum += steps(lane_seq(c, b, s));
    r.sum = wave_sum(sum) * c.H;
    return r;
}

// The cut of worker's steps where each has `per` of the total.
template <class B, class F>
__device__ inline Cut cut_at(const KvCache& c, const B& b, const Total& total, int per, int worker, int lane,
                             F steps) {
    Cut r;
    r.per = per;
    r.at = min(static_cast<int64_t>(worker) * r.per, static_cast<int64_t>(total.sum));
    r.end = min(r.at + r.per, total.sum);
    if (r.at >= r.end) return r;
    int base = 0;
    for (int x = 0;; x += 64) {
        const KvSeq s = x ? lane_seq(c, b, x + lane) : total.s;
        const int n = x ? steps(s) : total.steps;
        int in = n;  // inclusive sum
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(in, o);
            if (lane >= o) in += y;
        }
        const uint64_t hit = __ballot((base + in) * c.H > r.at);
        if (hit) {
            const int k = __builtin_ctzll(hit);
            r.seq = x + k;
            r.first = (base + __builtin_amdgcn_readlane(in - n, k)) * c.H;
            r.s.row = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(s.row), k));
            r.s.q = __builtin_amdgcn_readlane(s.q, k);
            r.s.n = __builtin_amdgcn_readlane(s.n, k);
            r.s.ok = __builtin_amdgcn_readlane(s.ok, k);
            r.s.from = kParts<B> ? __builtin_amdgcn_readlane(s.from, k) : 0;
            return r;
        }
        base += __builtin_amdgcn_readlane(in, 63);
    }
}

// Per sequence and head: the wave that begins it, and how many more have parts.
template <int D, int NT>
__device__ inline int2* joins_of(const KvAttend& a, const Plan& p) {
    return reinterpret_cast<int2*>(a.work + (int64_t(2) << p.log_workers) * (NT * 16) * (D + 2));
}

// Rows up to which a wave reads the cache for itself.  Two column tiles of 256-wide
// heads do not fit its registers: 32 sequences of 8000 tokens, 32 rows, 162 us so and
// 111 us through LDS.
constexpr int few_rows(int D) { return D == 256 ? 16 : 32; }

// Streaming waves on a SIMD: two hide each other's latencies as long as a wave's
// sums, operands and loads in flight fit half of its registers.  Four contexts of
// 130 k in 4 bits: one 123 us, two 90, four, which spill, 145; 32 sequences of 8000, 64-wide
// heads: 67, 49, 57; 256-wide ones: one 105, two, which spill, 169.
template <int D, int NT>
constexpr int kStreamWaves = D * NT >= 256 ? 1 : 2;

template <int BITS, int D, int NT>
__global__ __launch_bounds__(256, (kStreamWaves<D, NT>)) void kv_stream_kernel(KvCache c, KvBatch b, KvAttend a, Plan p) {
    __shared__ __align__(16) float sc[4][192];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int worker = blockIdx.x * 4 + wave;
    auto steps = [&](const KvSeq& s) {
        int lo, hi;
        return steps_of(s, a, &lo, &hi);
    };
    const Total total = all_steps(c, b, lane, steps);
    const Cut cut = cut_at(c, b, total, max(kLeast, (total.sum + (1 << p.log_workers) - 1) >> p.log_workers),
                           worker, lane, steps);
    if (cut.at >= cut.end) return;
    int at = cut.at;
    Share w;
    w.seq = cut.seq;
    w.split = 0;
    w.r0 = 0;
    w.s = cut.s;
    int lo, hi, n = steps_of(w.s, a, &lo, &hi);
    w.head = (at - cut.first) / n;
    int from = (at - cut.first) % n;
    while (true) {
        const int to = min(n, from + (cut.end - at));
        if (from == 0 && lane == 0)
            joins_of<D, NT>(a, p)[w.seq * c.H + w.head] = int2{worker, (at + n - 1) / cut.per - worker};
        w.rn = w.s.q * a.G;
        if (!w.s.ok) {
            fail_rows<D>(w, a, lane, 64);
        } else {
            span_of(w, a);
            w.lo = lo + from * kStep;
            w.hi = min(hi, lo + to * kStep);
            Rows<BITS, D, NT> rows;
            Stream<BITS, D, NT> st(c, b, w, lane);
            rows.start(w, a, 0, lane);
            st.open(w.lo, kStep);
            float own[NT];
            const float big = rows.largest(a, own);
            const float f = rows.scale(a, big, own) * (a.scale * kLog2e);
            st.run(rows, w.lo, kStep, f, sc[wave]);
            if (from == 0 && to == n)
                finish<BITS, D, NT>(w, a, 0, lane, rows);
            else
                keep<D, NT>(a.work, 2 * worker + (from == 0), 2 << p.log_workers, w.rn, lane,
                            rows.o, rows.m, rows.l);
        }
        at += to - from;
        if (at >= cut.end) return;
        from = 0;
        if (++w.head == c.H) {
            w.head = 0;
            do {
                w.s = kv_seq(b, ++w.seq, c.shift);
                n = steps_of(w.s, a, &lo, &hi);
            } while (n == 0);
        }
    }
}

// Many rows: 16 NC of them a wave, W waves.  A step's keys and values are turned to
// float16 once for the workgroup, in LDS in the order in which the operands are read
// (16 bytes a lane, consecutive), while the next step's bytes are on their way into
// registers.
// What bounds it are the vector and the matrix instructions of a SIMD's two waves,
// which overlap little: 8192 tokens over 36193, 32 heads of 128 on 8, 8 bits, 4.7 to
// 5.0 ms on different cards, 923 to 861 TFLOP/s (a large float16 product reaches 1343), the
// matrix cores 37% busy, the vector units 54%, LDS 35%.  At 4096 tokens over 16096 (922
// TFLOP/s) a copy of it without the exponentials reaches 1237, without turning codes to
// float16 1066, without either 1483.
// Two column tiles a wave: with one a step in LDS serves half as many rows (614
// TFLOP/s), with three and four the registers spill (564, 614).  256-wide heads: LDS
// holds one workgroup, so it has eight waves of one tile (835; four waves of two 604).
// A workgroup's LDS: kf [buffer][tile][product][lane], vf [buffer][half][tile][lane].
#define JHQ_MANY_LDS(BITS, D, W)                                    \
    __shared__ __align__(16) h8 kf[2][4 * Dim<BITS, D>::KS * 64];   \
    __shared__ __align__(16) h8 vf[2][2 * Dim<BITS, D>::DT * 64];   \
    __shared__ __align__(16) float sc[2][192];                      \
    __shared__ float bigs[W]

// Steps that many_rows has on their way.
template <class X, int BITS, int D, int NC, int W>
constexpr int ahead_of = 1;

// A workgroup's share: the block x of a launch, or what share_of() else is overloaded for, which then
// keeps the rows itself.
template <int BITS, int D, int NC, int W, class B, class X>
__device__ inline void many_rows(const KvCache& c, const B& b, const KvAttend& a, const Plan& p,
                                 const X& x, h8 (&kf)[2][4 * Dim<BITS, D>::KS * 64],
                                 h8 (&vf)[2][2 * Dim<BITS, D>::DT * 64], float (&sc)[2][192],
                                 float (&bigs)[W]) {
    using M = Dim<BITS, D>;
    using K = typename KeyReg<M::LB>::type;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int g = lane >> 4, r = lane & 15;
    const Share w = share_of(c, b, a, p, x);
    if (!w.any) return;
    if (!w.s.ok) {
        if (w.split == 0) fail_rows<D>(w, a, threadIdx.x, 64 * W);
        return;
    }
    if (w.split && w.lo >= w.hi) return;  // the join knows which parts there are

    Where<BITS, D> where(c, b, w, lane);
    if (w.lo < w.hi) where.look(w.lo);
    Rows<BITS, D, NC> rows;
    const int r0 = w.r0 + wave * NC * 16;
    rows.start(w, a, r0, lane);
    // Four waves stage a tile of keys and every fourth tile of values each; of eight,
    // the first four take the keys, the others the values.
    constexpr int VT = (M::ET + 3) / 4;
    const int part = wave & 3;
    const bool has_keys = W == 4 || wave < 4, has_values = W == 4 || wave >= 4;
    // Steps on their way into registers.
    constexpr int S = ahead_of<X, BITS, D, NC, W>;
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, S - 1> Last;
    K krs[S][M::NU];
    u4 vrs[S][VT];
    float kss[S], vss[S];
    bool deads[S], losts[S];
#pragma unroll
    for (int z = 0; z < S; z++) kss[z] = vss[z] = 0, deads[z] = losts[z] = true;
    auto fetch = [&](int j, auto slot) {
        constexpr int z = decltype(slot)::value;
        K(&kr)[M::NU] = krs[z];
        u4(&vr)[VT] = vrs[z];
        float &ks = kss[z], &vs = vss[z];
        bool &dead = deads[z], &lost = losts[z];
        const uint8_t *k, *v;
        const float* s;
        where.find(j, k, v, s);
        const bool none = where.pv < 0;
        // before the codes: waiting for a page then is not waiting for them
        if (S > 1 && j + kStep < w.hi) where.look(j + kStep);
        if (has_keys) {
#pragma unroll
            for (int u = 0; u < M::NU; u++)
                kr[u] = *reinterpret_cast<const K*>(k + part * (4 * M::ROW) + u * 256);
        }
        if (has_values) {
#pragma unroll
            for (int t = 0; t < VT; t++)
                if (M::ET % 4 == 0 || t * 4 + part < M::ET)
                    vr[t] = *reinterpret_cast<const u4*>(v + (t * 4 + part) * 256);
        }
        if (wave == W - 4) {
            ks = s[0];
            vs = s[1 << c.shift];
            dead = j + lane >= w.s.n;
            lost = none;
        }
        if (S == 1 && j + kStep < w.hi) where.look(j + kStep);
    };
    if (w.lo < w.hi) fetch(w.lo, Zero());
    if (S > 1 && w.lo + kStep < w.hi) fetch(w.lo + kStep, Last());
    float own[NC];
    float big = rows.largest(a, own);
    if (lane == 0) bigs[wave] = big;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; x++) big = fmaxf(big, bigs[x]);
    const float f = rows.scale(a, big, own) * (a.scale * kLog2e);
    auto stage = [&](int buf, auto slot) {
        constexpr int z = decltype(slot)::value;
        K(&kr)[M::NU] = krs[z];
        u4(&vr)[VT] = vrs[z];
        const float ks = kss[z], vs = vss[z];
        const bool dead = deads[z], lost = losts[z];
        if (has_keys) {
#pragma unroll
            for (int o = 0; o < M::LB / 8; o++) {
                const uint32_t x = kr[o >> 1][(o & 1) * 2], y = kr[o >> 1][(o & 1) * 2 + 1];
                if constexpr (BITS == 8) {
                    kf[buf][(part * M::KS + o) * 64 + lane] = half8(x, y);
                } else {
                    h8 lo, hi;
                    half4(x, y, lo, hi);
                    kf[buf][(part * M::KS + 2 * o) * 64 + lane] = lo;
                    kf[buf][(part * M::KS + 2 * o + 1) * 64 + lane] = hi;
                }
            }
        }
        if (has_values) {
#pragma unroll
            for (int t = 0; t < VT; t++) {
                const int e = t * 4 + part;
                if (M::ET % 4 != 0 && e >= M::ET) continue;
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
                    if constexpr (BITS == 8) {
                        vf[buf][(kk * M::DT + e) * 64 + lane] = half8(vr[t][2 * kk], vr[t][2 * kk + 1]);
                    } else {
                        h8 lo, hi;
                        half4(vr[t][2 * kk], vr[t][2 * kk + 1], lo, hi);
                        vf[buf][(kk * M::DT + e) * 64 + lane] = lo;
                        vf[buf][(kk * M::DT + e + M::ET) * 64 + lane] = hi;
                    }
                }
            }
        }
        if (wave == W - 4) token_terms(ks, vs, f, dead, lost, sc[buf] + lane);
    };
    int buf = 0;
    if (w.lo < w.hi) stage(0, Zero());
    const bool uneven = __syncthreads_or(rows.uneven);
    auto step = [&](int j, int buf, auto uneven) {
        const bool masked = j < w.full_lo || j + kStep > w.full_hi;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            f4 s[NC][2];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int q = 0; q < M::KS; q++) {
                    const h8 x = kf[buf][((hf * 2 + t) * M::KS + q) * 64 + lane];
#pragma unroll
                    for (int k = 0; k < NC; k++)
                        s[k][t] = mfma(x, rows.q[k][q], q ? s[k][t] : f4{0, 0, 0, 0});
                }
            h8 pr[NC];
            rows.weigh(s, sc[buf], lane, j, hf, masked, uneven, pr);
#pragma unroll
            for (int t = 0; t < M::DT; t++) {
                const h8 v = vf[buf][(hf * M::DT + t) * 64 + lane];
#pragma unroll
                for (int k = 0; k < NC; k++) rows.o[k][t] = mfma(v, pr[k], rows.o[k][t]);
            }
        }
    };
    // In parts, tiles may have few rows: waves without one only bring the others their operands.
    const bool rows_here = std::is_same<X, uint32_t>::value || r0 < w.r0 + w.rn;
    auto steps = [&](auto uneven) {
        for (int j = w.lo; j < w.hi; j += kStep, buf ^= 1) {
            if (j + kStep < w.hi) fetch(j + kStep, Zero());
            if (rows_here) step(j, buf, uneven);
            if (j + kStep < w.hi) stage(buf ^ 1, Zero());
            __syncthreads();
        }
    };
    auto two = [&](int j, auto p) {  // a step whose buffer and slot are p
        constexpr int z = decltype(p)::value;
        if (j + 2 * kStep < w.hi) fetch(j + 2 * kStep, p);
        if (rows_here) step(j, z, uneven);
        if (j + kStep < w.hi) stage(z ^ 1, std::integral_constant<int, S - 1 - z>());
        __syncthreads();
    };
    // A loop of its own for the rare tile, as a branch in it costs the others 3% (4096
    // tokens over 16096: 1053 and 1024 us); but two loops cost 64-wide heads the third
    // wave of a SIMD (753 and 776 us).
    if constexpr (S > 1) {
        for (int j = w.lo; j < w.hi; j += 2 * kStep) {
            two(j, Zero());
            if (j + kStep < w.hi) two(j + kStep, Last());
        }
    } else if constexpr (D == 64 || !std::is_same<X, uint32_t>::value)
        steps(uneven);
    else if (uneven)
        steps(std::true_type());
    else
        steps(std::false_type());
    rows.join();
    if constexpr (!std::is_same<X, uint32_t>::value) {
        x.keep(w, a, r0, lane, rows);
        return;
    }
    if (w.alone) return finish<BITS, D, NC>(w, a, r0, lane, rows);
#pragma unroll
    for (int k = 0; k < NC; k++) {
        const int row = r0 + k * 16 + r;
        if (row >= w.r0 + w.rn) continue;
        int64_t q;
        const int64_t o = w.split * p.rows + row_of(w, a, row, &q);
#pragma unroll
        for (int t = 0; t < M::DT; t++)
            *reinterpret_cast<f4*>(a.work + o * D + t * 16 + g * 4) = rows.o[k][t];
        if (g == 0) {
            float* const ml = a.work + p.nsplit * p.rows * D + o * 2;
            ml[0] = rows.m[k];
            ml[1] = rows.l[k];
        }
    }
}

template <int BITS, int D, int NC, int W>
__global__ __launch_bounds__(64 * W, W == 8 || D < 256 ? 2 : 1)
void kv_many_kernel(KvCache c, KvBatch b, KvAttend a, Plan p) {
    JHQ_MANY_LDS(BITS, D, W);
    many_rows<BITS, D, NC, W>(c, b, a, p, static_cast<uint32_t>(blockIdx.x), kf, vf, sc, bigs);
}

}  // namespace
}  // namespace jhq
