// kv_attend.hip — attention of new tokens over the quantised key/value cache: what joins the parts of
// rows, the rules that choose the kernels, and the launches.  The arithmetic and the kernels are in kv_attend.h.
#include "kv_attend.h"

namespace jhq {
namespace {

// Adds the parts of rows; latency bounds it.  Workgroups go over sequences of max_q tokens each
// or, where those are many more than the call's rows (new token, query head), over the rows, whose
// sequence a search of cu_q finds: 2048 tokens beside 63 single ones, 8000 each, 32 heads on 8
// of 128, 895 us a call in the first way and 662 in the second; 64 single tokens in the first
// lines of arrays of 65536, 109 and 701.  NT > 0: parts of kv_stream_kernel,
// often many: a thread has 4 elements of every fourth part of a row.  NT = 0: parts of
// kv_many_kernel, few parts and more rows: a thread has all of its elements' parts.
template <int NT>
constexpr int kJoinSplit = NT ? 4 : 1;
template <int D, int NT>
constexpr int kJoinRows = 1024 / D / kJoinSplit<NT>;  // rows of a workgroup

template <int D, int NT>
__global__ __launch_bounds__(256) void kv_join_kernel(KvCache c, KvBatch b, KvAttend a, Plan p) {
    constexpr int T = D / 4, R = kJoinRows<D, NT>, Y = kJoinSplit<NT>;
    constexpr int WR = 64 > Y * T ? 64 / (Y * T) : 1;  // rows of a wave
    __shared__ __align__(16) float acc[R][Y][D];
    __shared__ float ml[R][Y][2];
    const int t = threadIdx.x % T, y = threadIdx.x / T % Y, r = threadIdx.x / (Y * T);
    const int x = blockIdx.x * R + r;
    const int tok = x / a.heads, h = x - tok * a.heads;
    int seq = 0, i = 0;
    if (p.per) {
        seq = tok / p.per;
        i = tok - seq * p.per;
    } else {
        const int first = __builtin_amdgcn_readfirstlane(x);
#pragma unroll
        for (int k = 0; k < WR; k++) {
            // a wave's rows are mostly one token's
            const int mine = (first + k) / a.heads;
            if (k && mine == (first + k - 1) / a.heads) continue;
            const int s = last_at_most(b.n_seq, mine, [&](int j) { return b.cu_q[j]; });
            if (mine <= tok) seq = s;
        }
    }
    int n = 0;            // parts
    int64_t row = 0;      // of the output
    int64_t slot = 0, next = 0;  // the first part's row, and from one to the next
    int64_t jump = 0;     // added from the second on
    bool sees = false;
    KvSeq s = {0, 0, 0, false};
    if (seq < b.n_seq) s = kv_seq(b, seq, c.shift);
    if (!p.per) i = static_cast<int>(tok - s.row);
    if (s.ok && i >= 0 && i < s.q) {
        sees = sees_any(s, a, i);
        row = (s.row + i) * a.heads + h;
        if constexpr (NT > 0) {
            const int2 j = joins_of<D, NT>(a, p)[seq * c.H + h / a.G];
            n = j.y ? j.y + 1 : 0;  // one wave had it all and has written it
            slot = static_cast<int64_t>(2 * j.x + 1) * (NT * 16) + i * a.G + h % a.G;
            next = 2 * NT * 16;
            jump = -NT * 16;
        } else {
            // as in share_of
            const int tile = (i * a.G + h % a.G) / p.tile;
            const int last = min((tile + 1) * p.tile, s.q * a.G) - 1;
            const int from = see_lo(s, a, tile * p.tile / a.G) / kStep * kStep;
            const int hi = see_hi(s, a, last / a.G);
            // a tile of one part has been written already
            n = hi - from > p.chunk ? (hi - from + p.chunk - 1) / p.chunk : 0;
            slot = row;
            next = p.rows;
        }
    }
    const float* const stats = a.work + (NT > 0 ? (int64_t(2) << p.log_workers) * (NT * 16) * D
                                                : p.nsplit * p.rows * D);
    float m = kNone, l = 0.0f;
    f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int k = y; k < n; k += Y) {
        const int64_t at = slot + k * next + (k ? jump : 0);
        const float2 st = *reinterpret_cast<const float2*>(stats + at * 2);
        const f4 v = *reinterpret_cast<const f4*>(a.work + at * D + t * 4);
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
    if (y || n == 0) return;
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
    store4(a, row * D + t * 4, o * inverse_of(l, sees));
    if (a.lse && t == 0) a.lse[row] = lse_of(m, l, sees);
}

// What a call runs: 16 or 32 rows from registers (short or streaming), or tiles of 64 or
// 128 rows through LDS.  At 32 rows the former takes 71 us and the latter 76 for 64
// sequences of 8000 tokens on 2 heads of 128 in 8 bits, 61 and 70 in 4, 37 and 54 with heads
// of 64.
enum class Path { kShort, kStream, kMany };
struct Choice {
    Path path;
    int nc;     // column tiles of a wave
    int waves;  // of a workgroup of many rows
    Plan p;
    int64_t work;  // bytes, -1: more than 2^50
};

Choice choose(const KvCache& c, const KvBatch& b, int D, int G, int window) {
    Choice r;
    Plan& p = r.p;
    const int64_t rows = static_cast<int64_t>(b.max_q) * G;
    const int64_t span = window ? std::min<int64_t>(b.max_kv, static_cast<int64_t>(window) + b.max_q + kStep)
                                : b.max_kv;
    // the streaming kernel numbers steps with an int
    const bool counted = static_cast<int64_t>(b.n_seq) * c.H * (span / kStep + 2) < INT32_MAX / 2;
    r.path = rows > few_rows(D) ? Path::kMany
             : span <= kShortSpan ? Path::kShort : counted ? Path::kStream : Path::kMany;
    r.nc = r.path == Path::kMany ? (rows <= 64 ? 1 : 2) : (rows <= 16 ? 1 : 2);
    r.waves = r.path == Path::kMany && D == 256 && r.nc == 2 ? 8 : 4;
    if (r.waves == 8) r.nc = 1;
    p.tile = r.path == Path::kMany ? r.nc * 16 * r.waves : r.nc * 16;
    p.tiles = static_cast<int>((rows + p.tile - 1) / p.tile);
    // sequences whose rows overlap, which cu_q in order cannot say, may have more: the
    // tiles past these are not run
    p.real = std::min<int64_t>(static_cast<int64_t>(b.n_seq) * p.tiles,
                               b.n_tokens * G / p.tile + b.n_seq);
    p.rows = b.n_tokens * c.H * G;
    const int64_t all = static_cast<int64_t>(b.n_seq) * b.max_q;
    p.per = 2 * all > 3 * b.n_tokens ? 0 : b.max_q;
    p.nsplit = 1;
    p.chunk = 0;
    p.log_workers = 0;
    r.work = 0;
    if (r.path == Path::kStream) {
        p.log_workers = D * r.nc >= 256 ? 10 : 11;  // kStreamWaves on each of 1024 SIMDs
        r.work = (int64_t(2) << p.log_workers) * p.tile * (D + 2) * 4 +
                 static_cast<int64_t>(b.n_seq) * c.H * 8;
    } else if (r.path == Path::kMany) {
        // workgroups without a split: no more tiles than the rows fill
        const int64_t tiles = p.real * c.H;
        const int64_t seen = window ? std::min<int64_t>(b.max_kv, static_cast<int64_t>(window) +
                                                                      p.tile / G + 2 + kStep)
                                    : b.max_kv;
        // Parts only as far as the tiles do not fill the chip with two on each of 256 CUs:
        // 16 sequences of 8000 tokens, 64 rows on each of 8 heads: parts up to 256 workgroups
        // 115 us, 512 81, 1024 89, 2048 104; a prompt of 2999 tokens, where 768 tiles need
        // none: 120, and 152 with parts up to 1024.
        const int64_t parts = std::max<int64_t>(1, (512 + tiles - 1) / tiles);
        int64_t chunk = std::max<int64_t>(512, (seen + parts - 1) / parts);
        // Long contexts beyond that where the last round of workgroups leaves a tenth of the places
        // empty: a part of 4096 tokens or more outweighs its place in the join.  2500 tokens
        // over 32500, 32 heads on 8 of 128: 2027 us without, 1467 with; on 8 of 256 3683, 3237; 16
        // heads of 64, 4 bits, 561, 490; 64 x 10 to 100 over 9000 of the latter 570, 482.  Where
        // rounds are whole it costs: 2 x 1000 over 21000, 8 heads on 2 of 256, 450 without and 526
        // with; 4096 over 16096, 32 on 8 of 128, 1021, 1115.  Tiles are counted as the bounds allow:
        // where ragged lengths have fewer, it can be wrong (100 x 1 to 40 over 6000, 32 on 8 of
        // 128: 551, 579).
        const bool three = D == 64 && c.codes >> c.shift == 32;  // workgroups of a CU: 4 bits
        const int64_t places = D == 256 ? 256 : three ? 768 : 512;
        const int64_t groups = tiles * ((seen + chunk - 1) / chunk);
        const int64_t last = (groups + places - 1) / places * places;
        if (10 * groups < 9 * last) {
            const int64_t finer = (4 * places + tiles - 1) / tiles;
            chunk = std::min(chunk, std::max<int64_t>(4096, (seen + finer - 1) / finer));
        }
        chunk = (chunk + kStep - 1) / kStep * kStep;
        p.nsplit = static_cast<int>(std::max<int64_t>(1, (seen + chunk - 1) / chunk));
        if (p.nsplit > 1) {
            p.chunk = static_cast<int>(chunk);
            const __int128 work = static_cast<__int128>(p.nsplit) * p.rows * (D + 2) * 4;
            r.work = work > int64_t(1) << 50 ? -1 : static_cast<int64_t>(work);
        }
    }
    return r;
}

template <int BITS, int D>
hipError_t launch(const KvCache& c, const KvBatch& b, const KvAttend& a, const Choice& ch,
                  hipStream_t s) {
    const Plan& p = ch.p;
    // a launch has 2^32 threads
    const int64_t out = p.per ? static_cast<int64_t>(b.n_seq) * p.per * a.heads : p.rows;
    const int64_t blocks = ch.path == Path::kStream ? (1 << p.log_workers) / 4
                                                    : c.H * p.real * p.nsplit;
    const int jrows = ch.path == Path::kMany ? kJoinRows<D, 0> : kJoinRows<D, 1>;
    const int64_t joins = ch.path == Path::kStream || p.nsplit > 1 ? (out + jrows - 1) / jrows : 0;
    if (blocks >= 1 << 23 || joins >= 1 << 23) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks)), jgrid(static_cast<unsigned>(joins));
    switch (ch.path) {
        case Path::kShort:
            if (ch.nc == 1)
                kv_short_kernel<BITS, D, 1, kShortWaves<D>>
                    <<<grid, 64 * kShortWaves<D>, 0, s>>>(c, b, a, p);
            else if constexpr (few_rows(D) > 16)
                kv_short_kernel<BITS, D, 2, kShortWaves<D>>
                    <<<grid, 64 * kShortWaves<D>, 0, s>>>(c, b, a, p);
            break;
        case Path::kStream:
            if (ch.nc == 1)
                kv_stream_kernel<BITS, D, 1><<<grid, 256, 0, s>>>(c, b, a, p);
            else if constexpr (few_rows(D) > 16)
                kv_stream_kernel<BITS, D, 2><<<grid, 256, 0, s>>>(c, b, a, p);
            break;
        case Path::kMany:
            if (ch.nc == 1 && ch.waves == 4)
                kv_many_kernel<BITS, D, 1, 4><<<grid, 256, 0, s>>>(c, b, a, p);
            else if constexpr (D == 256)
                kv_many_kernel<BITS, D, 1, 8><<<grid, 512, 0, s>>>(c, b, a, p);
            else
                kv_many_kernel<BITS, D, 2, 4><<<grid, 256, 0, s>>>(c, b, a, p);
            break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || joins == 0) return e;
    if (ch.path == Path::kMany)
        kv_join_kernel<D, 0><<<jgrid, 256, 0, s>>>(c, b, a, p);
    else if (ch.nc == 1)
        kv_join_kernel<D, 1><<<jgrid, 256, 0, s>>>(c, b, a, p);
    else if constexpr (few_rows(D) > 16)
        kv_join_kernel<D, 2><<<jgrid, 256, 0, s>>>(c, b, a, p);
    return hipGetLastError();
}

}  // namespace

int64_t kv_attend_work(const KvCache& c, const KvBatch& b, int D, int G, int window) {
    return choose(c, b, D, G, window).work;
}

hipError_t kv_attend(const KvCache& c, const KvBatch& b, int bits, int D, const KvAttend& a,
                     hipStream_t s) {
    const Choice p = choose(c, b, D, a.G, a.window);
    if (bits == 8)
        return D == 64 ? launch<8, 64>(c, b, a, p, s)
                       : D == 128 ? launch<8, 128>(c, b, a, p, s) : launch<8, 256>(c, b, a, p, s);
    return D == 64 ? launch<4, 64>(c, b, a, p, s)
                   : D == 128 ? launch<4, 128>(c, b, a, p, s) : launch<4, 256>(c, b, a, p, s);
}

}  // namespace jhq
