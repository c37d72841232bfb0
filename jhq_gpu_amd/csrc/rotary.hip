// rotary.hip — queries and keys turned to their positions (jhq_k_rotary).
//
// Mathematics.  Pair (x0, x1) of a token at position p becomes A (x0 cos a - x1 sin a, x1 cos a
// + x0 sin a), a = p f; the angle's arithmetic is in rotary.h.  The inverse (a turned to -a) is the
// gradient: it is the transposed matrix.
//
// Layout.  A wave's lanes are W columns of a head's units times 64 / W rows (a token's heads); a
// unit is E pairs: two runs of E elements, half of the pairs' elements apart, so that neighbouring lanes
// have neighbouring runs (single pairs side by side are neighbours themselves).  A lane keeps its column,
// so it has its E angles' sines and cosines once for all of a token's heads.
//
// HBM-bound: 13003 tokens of 40 heads of 128 in float16, side by side, 208 MB in 43.8 us, 4.75 TB/s (a
// large copy moves 4.8; 50.5 with a unit's runs beside each other); 8191 of 12 of 256 in float32, a quarter
// turned, 41 us, 4.9 TB/s.  Single tokens are a launch: 3.2 us, 5.8 a call.
#include "kvcache.h"
#include "rotary.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

// Defined in jhq_capi.hip: sets the thread-local message jhq_last_error returns.
int jhq_set_error(int code, const char* msg);

namespace jhq {
namespace {

struct Turn {
    Rotary r;
    KvRows x;
    void* out;
    int64_t out_tok, out_head;
    int64_t n_tokens;
    int heads;
    const void* pos;  // of each token, or null: n - q + i of the batch's sequences
    int wide;         // 64-bit positions
    const int32_t *kv_len, *cu_q;
    int n_seq;
    // how the work is cut
    int pairs, cols;  // columns of a head that turn, and all of them (the rest is copied)
    int width;        // columns at once, W
    int hg, tg;       // heads and tokens at once: hg * tg * W <= 64
    int splits, per;  // parts of a token's heads, heads of each
    int blocks;       // of W columns
    uint32_t units;   // waves that have work
};

template <int BYTES>
struct Raw {
    typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4)));
};
template <>
struct Raw<4> {
    typedef uint32_t type;
};
template <>
struct Raw<2> {
    typedef uint16_t type;
};

template <int DT, int E>
struct Run {
    static constexpr int SIZE = DT == JHQ_F32 ? 4 : 2;
    typedef typename Raw<E * SIZE>::type type;
    typedef typename std::conditional<DT == JHQ_F32, float, uint16_t>::type el;
    __device__ static type load(const void* p, int64_t i) {
        return *reinterpret_cast<const type*>(static_cast<const el*>(p) + i);
    }
    __device__ static void store(void* p, int64_t i, type v) {
        *reinterpret_cast<type*>(static_cast<el*>(p) + i) = v;
    }
    __device__ static void open(type v, float* x) {
        el e[E];
        __builtin_memcpy(e, &v, sizeof v);
#pragma unroll
        for (int i = 0; i < E; i++) {
            if constexpr (DT == JHQ_F32)
                x[i] = e[i];
            else if constexpr (DT == JHQ_BF16)
                x[i] = __uint_as_float(static_cast<uint32_t>(e[i]) << 16);
            else
                x[i] = static_cast<float>(__builtin_bit_cast(_Float16, e[i]));
        }
    }
    __device__ static type close(const float* x) {
        el e[E];
#pragma unroll
        for (int i = 0; i < E; i++) {
            if constexpr (DT == JHQ_F32)
                e[i] = x[i];
            else if constexpr (DT == JHQ_BF16)
                e[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[i]));
            else
                e[i] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[i]));
        }
        type v;
        __builtin_memcpy(&v, e, sizeof v);
        return v;
    }
};

// The position of token t of the batch; false where no sequence has the row.  The wave asks for one
// token.
__device__ inline bool place_of(const Turn& a, int64_t t, int64_t* pos) {
    const int s = last_at_most(a.n_seq, t, [&](int j) { return a.cu_q[j]; });
    const int64_t c0 = a.cu_q[s], c1 = a.cu_q[s + 1];
    *pos = a.kv_len[s] - (c1 - t);
    return t >= c0 && t < c1;
}

// Heads in flight: 13003 tokens of 40 heads of 128 in float16 43.8 us with two, 46.0 with four, of 8
// heads in bfloat16 11.6 and 12.6.
constexpr int kDeep = 2;

template <int DT, int E, bool SIDE>
__global__ __launch_bounds__(256) void rotary_kernel(Turn a) {
    using R = Run<DT, E>;
    const int lane = threadIdx.x & 63;
    uint32_t u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= a.units) return;
    const int blk = u % static_cast<uint32_t>(a.blocks);
    u /= static_cast<uint32_t>(a.blocks);
    const int split = u % static_cast<uint32_t>(a.splits);
    const int64_t t0 = static_cast<int64_t>(u / static_cast<uint32_t>(a.splits)) * a.tg;
    const int c = blk * a.width + lane % a.width, row = lane / a.width;
    const int tk = row / a.hg;
    const int64_t t = t0 + tk;
    bool live = c < a.cols && tk < a.tg && t < a.n_tokens;
    int64_t pos = 0;
    if (a.pos) {
        if (live)
            pos = a.wide ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
    } else {
        bool has = false;
        for (int k = 0; k < a.tg && t0 + k < a.n_tokens; k++) {
            int64_t p;
            const bool is = place_of(a, t0 + k, &p);
            if (tk == k) has = is, pos = p;
        }
        live = live && has;
    }
    if (!live) return;
    const bool turns = c < a.pairs;
    float co[E], si[E];
    if (turns) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            turn_of(a.r.turns[!SIDE || E == 1 ? c * E + e : (c * E + (2 * e < E ? 0 : a.r.rot / 2 - E)) / 2 + e], pos,
                    co[e], si[e]);
            co[e] *= a.r.amp;
            si[e] *= a.r.sign;
        }
    }
    // the unit's two runs
    int e0, e1;
    if (!turns) {
        e0 = a.r.rot + (c - a.pairs) * E;
        e1 = e0 + (a.cols - a.pairs) * E;
    } else if (SIDE && E == 1) {
        e0 = 2 * c;
        e1 = e0 + 1;
    } else {
        e0 = E * c;
        e1 = e0 + a.r.rot / 2;
    }
    const int end = min(a.heads, (split + 1) * a.per);
    const int64_t xb = t * a.x.tok, ob = t * a.out_tok;
    for (int h0 = split * a.per + row % a.hg; h0 < end; h0 += kDeep * a.hg) {
        typename R::type v[kDeep][2];
#pragma unroll
        for (int k = 0; k < kDeep; k++) {
            const int h = h0 + k * a.hg;
            if (h < end) {
                v[k][0] = R::load(a.x.p, xb + h * a.x.head + e0);
                v[k][1] = R::load(a.x.p, xb + h * a.x.head + e1);
            }
        }
#pragma unroll
        for (int k = 0; k < kDeep; k++) {
            const int h = h0 + k * a.hg;
            if (h >= end) break;
            if (turns) {
                float x[2 * E], y[2 * E];
                R::open(v[k][0], x);
                R::open(v[k][1], x + E);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    // side by side, a run has its pairs within itself
                    const int p = SIDE ? 2 * e : e, q = SIDE ? 2 * e + 1 : e + E;
                    y[p] = fmaf(x[p], co[e], -(x[q] * si[e]));
                    y[q] = fmaf(x[q], co[e], x[p] * si[e]);
                }
                v[k][0] = R::close(y);
                v[k][1] = R::close(y + E);
            }
            R::store(a.out, ob + h * a.out_head + e0, v[k][0]);
            R::store(a.out, ob + h * a.out_head + e1, v[k][1]);
        }
    }
}

// Launches kernels of E elements a run.
template <int DT, int E>
hipError_t launch(Turn& a, int head_dim, bool same, hipStream_t s) {
    a.pairs = a.r.rot / 2 / E;
    // the rest of a head stays where it is in place
    a.cols = a.pairs + (same ? 0 : (head_dim - a.r.rot) / (2 * E));
    a.width = std::min(a.cols, 64);
    a.blocks = (a.cols + a.width - 1) / a.width;
    const int rows = 64 / a.width;
    a.hg = std::min(a.heads, rows);
    a.tg = rows / a.hg;
    const int64_t tokens = (a.n_tokens + a.tg - 1) / a.tg;
    // a token's heads are split as far as waves do not fill the chip (two on a SIMD)
    const int most = (a.heads + a.hg - 1) / a.hg;
    const int64_t want = (2048 + tokens * a.blocks - 1) / (tokens * a.blocks);
    const int times = (most + std::min<int64_t>(want, most) - 1) / static_cast<int>(std::min<int64_t>(want, most));
    a.per = times * a.hg;
    a.splits = (a.heads + a.per - 1) / a.per;
    const int64_t units = tokens * a.splits * a.blocks, blocks = (units + 3) / 4;
    if (blocks >= 1 << 23) return hipErrorInvalidValue;
    a.units = static_cast<uint32_t>(units);
    if (a.r.interleaved)
        rotary_kernel<DT, E, true><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
    else
        rotary_kernel<DT, E, false><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
    return hipGetLastError();
}

// Runs of 16 bytes, of 8 or single elements: the longest that the head's parts are made of and
// that rows start on.
template <int DT>
hipError_t choose(Turn& a, int head_dim, bool same, hipStream_t s) {
    constexpr int SIZE = DT == JHQ_F32 ? 4 : 2;
    auto fits = [&](int e) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(a.x.p) | reinterpret_cast<uintptr_t>(a.out);
        return a.r.rot % (2 * e) == 0 && (same || (head_dim - a.r.rot) % (2 * e) == 0) &&
               p % (e * SIZE) == 0 && a.x.tok % e == 0 && a.x.head % e == 0 && a.out_tok % e == 0 &&
               a.out_head % e == 0;
    };
    if (fits(16 / SIZE)) return launch<DT, 16 / SIZE>(a, head_dim, same, s);
    if (fits(8 / SIZE)) return launch<DT, 8 / SIZE>(a, head_dim, same, s);
    return launch<DT, 1>(a, head_dim, same, s);
}

int bad(const std::string& msg) { return jhq_set_error(JHQ_EINVAL, msg.c_str()); }

int do_rotary(const jhq_rotary* r, const void* d_x, int64_t x_tok, int64_t x_head, int64_t n_tokens,
              int heads, int dtype, const void* d_pos, int pos_bytes, const jhq_kv_batch* b,
              int inverse, void* d_out, int64_t out_tok, int64_t out_head, void* stream) {
    const std::string wrong = rotary_wrong(r);
    if (!wrong.empty()) return bad(wrong);
    if (dtype != JHQ_F32 && dtype != JHQ_BF16 && dtype != JHQ_F16)
        return bad("rows must be JHQ_F32, JHQ_BF16 or JHQ_F16");
    if (n_tokens < 0 || n_tokens > INT32_MAX) return bad("n_tokens must be 0 .. 2^31 - 1");
    if (heads < 0 || heads > 1 << 20) return bad("heads must be 0 .. 2^20");
    if (inverse != 0 && inverse != 1) return bad("inverse must be 0 or 1");
    if ((d_pos != nullptr) == (b != nullptr) && n_tokens > 0)
        return bad("positions come from an array or from a batch");
    if (d_pos && pos_bytes != 4 && pos_bytes != 8) return bad("positions have 4 or 8 bytes");
    if (b) {
        if (b->n_tokens != n_tokens) return bad("the batch has another number of rows");
        if (b->n_seq < 0) return bad("negative size in the batch");
        if (b->n_seq > 0 && (!b->d_kv_len || !b->d_cu_q)) return bad("null array in the batch");
    }
    if (n_tokens == 0 || heads == 0 || (b && b->n_seq == 0)) return JHQ_OK;
    if (!d_x || !d_out) return bad("null rows or output");
    const bool same = d_x == d_out && x_tok == out_tok && x_head == out_head;
    Turn a = {};
    a.r = rotary_of(*r, inverse != 0);
    a.x = {d_x, x_tok, x_head};
    a.out = d_out;
    a.out_tok = out_tok;
    a.out_head = out_head;
    a.n_tokens = n_tokens;
    a.heads = heads;
    a.pos = d_pos;
    a.wide = pos_bytes == 8;
    if (b) {
        a.kv_len = b->d_kv_len;
        a.cu_q = b->d_cu_q;
        a.n_seq = b->n_seq;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == JHQ_F32    ? choose<JHQ_F32>(a, r->head_dim, same, s)
                         : dtype == JHQ_BF16 ? choose<JHQ_BF16>(a, r->head_dim, same, s)
                                             : choose<JHQ_F16>(a, r->head_dim, same, s);
    if (e == hipSuccess) return JHQ_OK;
    (void)hipGetLastError();  // reported here: not the next launch's
    if (e == hipErrorInvalidValue) return bad("rotary: more work than one launch holds");
    return jhq_set_error(e == hipErrorOutOfMemory ? JHQ_ENOMEM : JHQ_EDEVICE,
                         (std::string("rotary: ") + hipGetErrorString(e)).c_str());
}

}  // namespace

std::string rotary_wrong(const jhq_rotary* r) {
    if (!r) return "null rotary parameters";
    if (r->head_dim < 2 || r->head_dim > 1024 || r->head_dim % 2) return "head_dim must be even, 2 .. 1024";
    if (r->rot_dim < 2 || r->rot_dim > r->head_dim || r->rot_dim % 2)
        return "rot_dim must be even, 2 .. head_dim";
    if (r->interleaved != 0 && r->interleaved != 1) return "interleaved must be 0 or 1";
    if (!std::isfinite(r->amplitude)) return "amplitude must be finite";
    if (!r->d_turns || reinterpret_cast<uintptr_t>(r->d_turns) & 7)
        return "turns must be an array on 8 bytes";
    return "";
}

Rotary rotary_of(const jhq_rotary& r, bool inverse) {
    return {r.d_turns, r.rot_dim, r.interleaved, r.amplitude, inverse ? -r.amplitude : r.amplitude};
}

}  // namespace jhq

extern "C" int jhq_k_rotary(const jhq_rotary* r, const void* d_x, int64_t x_tok, int64_t x_head,
                            int64_t n_tokens, int heads, int dtype, const void* d_pos, int pos_bytes,
                            const jhq_kv_batch* batch, int inverse, void* d_out, int64_t out_tok,
                            int64_t out_head, void* stream) {
    try {
        return jhq::do_rotary(r, d_x, x_tok, x_head, n_tokens, heads, dtype, d_pos, pos_bytes, batch,
                              inverse, d_out, out_tok, out_head, stream);
    } catch (...) {  // no memory for a message
        return JHQ_ENOMEM;
    }
}
