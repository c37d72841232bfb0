// kv_attend.hip — attention of new tokens over the quantised key/value cache: what joins the parts of
// rows, and the launches.  Its arithmetic and its kernels are in kv_attend.h.
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
