// kv_shared.hip — attention of sequences in groups that share a prefix of the key/value cache.
//
// Mathematics.  The rows of a group (new tokens x query heads of a key head) all see all of the
// group's prefix, so over it they are the rows of one sequence, whose codes are read and
// turned once for all of them.  Over what stands behind the prefix every sequence is on its own.  Both
// passes are the kernels of kv_attend.h; of each a row has parts (maximum, sum, sums of values),
// and as softmax does not care in what order its sums are taken, joining all of them is the
// attention over all tokens:  m = max m_p, l = sum 2^(m_p - m) l_p, o = sum 2^(m_p - m) o_p / l.
#include "kv_attend.h"

namespace jhq {
namespace {

// A pass's parts, as the join finds them.
struct Source {
    Plan p;
    Path path;
    const float* work;
};

// The parts of a row: their number, the first one's place and the way to the others, sums of values
// and (maximum, sum).
struct Parts {
    int n;
    int64_t first, next, jump;
    const float *o, *ml;
    __device__ int64_t at(int k) const { return first + k * next + (k ? jump : 0); }
};

template <int D, class B>
__device__ inline Parts parts_of(const Source& x, const KvCache& c, const B& b, const KvAttend& a,
                                 const KvSeq& s, int seq, int i, int h) {
    const Plan& p = x.p;
    const int64_t row = (s.row + i) * a.heads + h;
    if (x.path == Path::kShort) return {1, row, 0, 0, x.work, x.work + p.rows * D};
    if (x.path == Path::kStream) {
        const int64_t slots = (int64_t(2) << p.log_workers) * p.tile;
        const float* const behind = x.work + slots * (D + 2);
        const int2 j = reinterpret_cast<const int2*>(behind)[seq * c.H + h / a.G];
        if (j.y == 0) {
            const float* const whole = behind + (static_cast<int64_t>(b.n_seq) * c.H + 1) / 2 * 4;
            return {1, row, 0, 0, whole, whole + p.rows * D};
        }
        return {j.y + 1, static_cast<int64_t>(2 * j.x + 1) * p.tile + i * a.G + h % a.G,
                2 * static_cast<int64_t>(p.tile), -static_cast<int64_t>(p.tile), x.work,
                x.work + slots * D};
    }
    // as in share_of
    const int tile = (i * a.G + h % a.G) / p.tile;
    const int last = min((tile + 1) * p.tile, s.q * a.G) - 1;
    const int from = see_lo(s, a, tile * p.tile / a.G) / kStep * kStep;
    const int hi = see_hi(s, a, last / a.G);
    const int n = p.nsplit > 1 && hi - from > p.chunk ? (hi - from + p.chunk - 1) / p.chunk : 1;
    return {n, row, p.rows, 0, x.work, x.work + p.nsplit * p.rows * D};
}

// Joins what the passes have of a row; latency and reading the parts bound it.  A thread has 4
// elements of every Y-th part.
template <int D, int Y>
__global__ __launch_bounds__(256) void kv_shared_join_kernel(KvCache c, KvOwn b, KvLead lead, KvAttend a,
                                                             Source ls, Source os) {
    constexpr int T = D / 4, R = 256 / (T * Y);
    constexpr int WR = 64 > Y * T ? 64 / (Y * T) : 1;  // rows of a wave
    __shared__ __align__(16) float acc[R][Y][D];
    __shared__ float ml[R][Y][2];
    const int t = threadIdx.x % T, y = threadIdx.x / T % Y, r = threadIdx.x / (Y * T);
    const int x = blockIdx.x * R + r;
    const int tok = x / a.heads, h = x - tok * a.heads;
    int seq = 0, grp = 0;
    const int first = __builtin_amdgcn_readfirstlane(x);
#pragma unroll
    for (int k = 0; k < WR; k++) {
        // a wave's rows are mostly one token's
        const int mine = (first + k) / a.heads;
        if (k && mine == (first + k - 1) / a.heads) continue;
        const int s = last_at_most(b.n_seq, mine, [&](int j) { return b.cu_q[j]; });
        const int g = last_at_most(lead.n_seq, mine, [&](int j) { return lead.cu_q[j]; });
        if (mine <= tok) seq = s, grp = g;
    }
    const KvSeq s = kv_seq(b, seq, c.shift);
    const int64_t i = tok - s.row;
    const bool has = x < os.p.rows && i >= 0 && i < s.q;
    bool ok = s.ok, sees = false;
    Parts A = {}, O = {};
    if (has && ok) {
        sees = sees_any(s, a, static_cast<int>(i));
        O = parts_of<D>(os, c, b, a, s, seq, static_cast<int>(i), h);
        const KvSeq w = kv_seq(lead, grp, c.shift);
        const int64_t li = tok - w.row;
        if (tok >= lead.cu_q[grp] && tok < lead.cu_q[grp + 1]) {
            ok = w.ok && li < w.q;
            if (ok) {
                KvAttend la = a;
                la.causal = 0;
                sees |= w.n > 0;
                A = parts_of<D>(ls, c, lead, la, w, grp, static_cast<int>(li), h);
            }
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
    if constexpr (Y > 1) {
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
    }
    if (!has) return;
    const int64_t row = static_cast<int64_t>(tok) * a.heads + h;
    const float bad = nan32();
    store4(a, row * D + t * 4, ok ? o * inverse_of(l, sees) : f4{bad, bad, bad, bad});
    if (a.lse && t == 0) a.lse[row] = ok ? lse_of(m, l, sees) : bad;
}

// What a call runs.
struct Both {
    bool shared;  // false: attention as without a prefix
    Choice lead, own;
    int64_t work;  // bytes, -1: more than 2^50
};

Both choose_both(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G) {
    Both r;
    r.shared = lead.n_seq > 0 && lead.max_kv > 0 && static_cast<int64_t>(b.max_q) * G < 128;
    if (!r.shared) {
        r.own = choose(c, b, D, G, 0);
        r.work = r.own.work;
        return r;
    }
    r.lead = choose(c, lead, D, G, 0, true);
    if (r.lead.work > 0) r.lead.work = (r.lead.work + 15) & ~int64_t(15);  // the other pass's lies behind
    r.own = choose(c, b, D, G, 0, true);
    r.work = r.lead.work < 0 || r.own.work < 0 ? -1 : r.lead.work + r.own.work;
    return r;
}

template <int BITS, int D, class B>
hipError_t pass(const KvCache& c, const B& b, const KvAttend& a, const Choice& ch, hipStream_t s) {
    const Plan& p = ch.p;
    const int64_t blocks = ch.path == Path::kStream ? (1 << p.log_workers) / 4 : c.H * p.real * p.nsplit;
    if (blocks >= 1 << 23) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks));
    switch (ch.path) {
        case Path::kShort:
            if (ch.nc == 1)
                kv_short_kernel<BITS, D, 1, kShortWaves<D>, B><<<grid, 64 * kShortWaves<D>, 0, s>>>(c, b, a, p);
            else if constexpr (few_rows(D) > 16)
                kv_short_kernel<BITS, D, 2, kShortWaves<D>, B><<<grid, 64 * kShortWaves<D>, 0, s>>>(c, b, a, p);
            break;
        case Path::kStream:
            if (ch.nc == 1)
                kv_stream_kernel<BITS, D, 1, B><<<grid, 256, 0, s>>>(c, b, a, p);
            else if constexpr (few_rows(D) > 16)
                kv_stream_kernel<BITS, D, 2, B><<<grid, 256, 0, s>>>(c, b, a, p);
            break;
        case Path::kMany:
            if (ch.nc == 1 && ch.waves == 4)
                kv_many_kernel<BITS, D, 1, 4, B><<<grid, 256, 0, s>>>(c, b, a, p);
            else if constexpr (D == 256)
                kv_many_kernel<BITS, D, 1, 8, B><<<grid, 512, 0, s>>>(c, b, a, p);
            else
                kv_many_kernel<BITS, D, 2, 4, B><<<grid, 256, 0, s>>>(c, b, a, p);
            break;
    }
    return hipGetLastError();
}

template <int BITS, int D>
hipError_t launch(const KvCache& c, const KvBatch& lead, const KvBatch& b, const KvAttend& a,
                  const Both& ch, hipStream_t s) {
    constexpr int Y = 4;
    const int64_t joins = (ch.own.p.rows + 256 / (D / 4 * Y) - 1) / (256 / (D / 4 * Y));
    if (joins >= 1 << 23) return hipErrorInvalidValue;
    KvLead lb;
    static_cast<KvBatch&>(lb) = lead;
    KvOwn ob;
    static_cast<KvBatch&>(ob) = b;
    ob.lead_cu = lead.cu_q;
    ob.lead_len = lead.kv_len;
    ob.n_lead = lead.n_seq;
    KvAttend la = a, oa = a;
    la.causal = 0;
    oa.work = a.work + ch.lead.work / 4;
    hipError_t e = pass<BITS, D>(c, lb, la, ch.lead, s);
    if (e == hipSuccess) e = pass<BITS, D>(c, ob, oa, ch.own, s);
    if (e != hipSuccess) return e;
    kv_shared_join_kernel<D, Y><<<static_cast<unsigned>(joins), 256, 0, s>>>(
        c, ob, lb, a, {ch.lead.p, ch.lead.path, la.work}, {ch.own.p, ch.own.path, oa.work});
    return hipGetLastError();
}

}  // namespace

int64_t kv_shared_work(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G) {
    return choose_both(c, lead, b, D, G).work;
}

hipError_t kv_attend_shared(const KvCache& c, const KvBatch& lead, const KvBatch& b, int bits, int D,
                            const KvAttend& a, hipStream_t s) {
    const Both p = choose_both(c, lead, b, D, a.G);
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
