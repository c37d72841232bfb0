// kvcache.hip — the quantised key/value cache: its entry points (jhq_kv_*,
// jhq_k_kv_*), quantising rows into it and reading them back.
//
// Both directions are copies with a few operations per element, bound by HBM.
// One wave takes a run of 16 tokens (32 where their codes are fewer than 64 x 16
// bytes) of one head, keys or values.  On the side of the rows a lane holds 8
// consecutive elements, D / 8 lanes a row, so that rows move 16 bytes a lane and
// a row's largest magnitude is a maximum over neighbouring lanes; on the side of
// the cache a lane holds 16 consecutive code bytes.  Between the two the codes
// pass through LDS, [piece][token][16 bytes]; values, which the cache holds
// token-minor, have their 16 x 16 byte tiles turned there.
#include "kvcache.h"
#include "rotary.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

// Defined in jhq_capi.hip: sets the thread-local message jhq_last_error returns.
int jhq_set_error(int code, const char* msg);

namespace jhq {
namespace {

constexpr int kWaves = 4;           // waves of a workgroup, each on its own
constexpr int kTilePitch = 272;     // bytes from one 16 x 16 tile to the next: 16 apart in the banks
constexpr float kFloor = 0x1p-60f;  // rows below it are held as zeros

// Sizes that follow from the bits and the head's elements.
template <int BITS, int D>
struct Run {
    static constexpr int ROW = D * BITS / 8;           // code bytes of a row
    static constexpr int NP = ROW / 16;                // pieces of it
    static constexpr int TW = ROW < 64 ? 32 : 16;      // tokens of a run
    static constexpr int CL = D / 8;                   // lanes of a row
    static constexpr int RI = 64 / CL, NI = TW / RI;   // rows at once; times
    static constexpr int OUT = TW * ROW / 16 / 64;     // 16-byte units of a lane
    static constexpr int LDS = TW / 16 * NP * kTilePitch;
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ inline float nan32() { return __uint_as_float(0x7fc00000u); }

// The values of 8 elements from element i on.
template <int DT, bool VEC>
__device__ inline void load8(const void* base, int64_t i, float* x) {
    if constexpr (DT == JHQ_F32) {
        const float* p = static_cast<const float*>(base) + i;
        if constexpr (VEC) {
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const float4 f = reinterpret_cast<const float4*>(p)[w];
                x[4 * w] = f.x, x[4 * w + 1] = f.y, x[4 * w + 2] = f.z, x[4 * w + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = p[j];
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + i;
        uint16_t h[8];
        if constexpr (VEC) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int j = 0; j < 4; j++) h[2 * j] = a[j] & 0xffff, h[2 * j + 1] = a[j] >> 16;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = p[j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            x[j] = DT == JHQ_BF16 ? __uint_as_float(static_cast<uint32_t>(h[j]) << 16)
                                  : static_cast<float>(__builtin_bit_cast(_Float16, h[j]));
    }
}

template <int DT>
__device__ inline float load1(const void* base, int64_t i) {
    if constexpr (DT == JHQ_F32) return static_cast<const float*>(base)[i];
    const uint16_t h = static_cast<const uint16_t*>(base)[i];
    return DT == JHQ_BF16 ? __uint_as_float(static_cast<uint32_t>(h) << 16)
                          : static_cast<float>(__builtin_bit_cast(_Float16, h));
}

template <int DT>
__device__ inline uint32_t round16(float f) {
    if constexpr (DT == JHQ_BF16)
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
    else
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
}

template <int DT, bool VEC>
__device__ inline void store8(void* base, int64_t i, const float* x) {
    if constexpr (DT == JHQ_F32) {
        float* p = static_cast<float*>(base) + i;
        if constexpr (VEC) {
#pragma unroll
            for (int w = 0; w < 2; w++)
                reinterpret_cast<float4*>(p)[w] =
                    make_float4(x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = x[j];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(base) + i;
        if constexpr (VEC) {
            u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++)
                o[j] = round16<DT>(x[2 * j]) | round16<DT>(x[2 * j + 1]) << 16;
            *reinterpret_cast<u32x4*>(p) = o;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = static_cast<uint16_t>(round16<DT>(x[j]));
        }
    }
}

// Orders a wave's LDS accesses before and after it (one wave: they execute in
// program order, the compiler only has to keep it).
__device__ inline void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Row i of m (4 bytes) becomes column i.
__device__ inline void transpose4(uint32_t m[4]) {
    const uint32_t a = __builtin_amdgcn_perm(m[1], m[0], 0x05010400);
    const uint32_t b = __builtin_amdgcn_perm(m[3], m[2], 0x05010400);
    const uint32_t c = __builtin_amdgcn_perm(m[1], m[0], 0x07030602);
    const uint32_t d = __builtin_amdgcn_perm(m[3], m[2], 0x07030602);
    m[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
    m[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    m[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
    m[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}

// Transposes a 16 x 16 byte tile in LDS in place, 16 lanes a tile: words by 4 x 4
// bytes.
__device__ inline void transpose16(uint8_t* tile, int lane) {
    const int r = (lane & 3) * 4, c = (lane >> 2 & 3) * 4;
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = *reinterpret_cast<const uint32_t*>(tile + (r + i) * 16 + c);
    wave_lds_fence();
    transpose4(m);
#pragma unroll
    for (int i = 0; i < 4; i++) *reinterpret_cast<uint32_t*>(tile + (c + i) * 16 + r) = m[i];
    wave_lds_fence();
}

// What one wave works on: a run of tokens from `first` (a multiple of 16), one
// head, keys or values.
struct Unit {
    KvSeq q;
    int seq, head, value;
    int first, lo;  // first token of the run; first new token (not below 0)
    bool any;
};

// The sequences' runs are numbered one after the other: sets of them each or, where lengths
// differ (SEARCH), from cu_q / TW + 2 seq on, which leaves floor(q / TW) + 2 at least for q new
// tokens that may begin and end inside a group, and is found by a search.  A prompt of 32768 tokens
// beside 511 single ones, 8 heads of 128, 8 bits: written in 2624 us with sets, 46 so; 64 prompts
// of 100 to 500: 24.5, 21.9.
template <int TW, bool SEARCH>
__device__ inline Unit unit_of(const KvCache& c, const KvBatch& b, int sets) {
    Unit r;
    uint32_t u = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    r.value = u & 1;
    u >>= 1;
    r.head = u % c.H;
    u /= c.H;
    int set;
    if constexpr (!SEARCH) {
        set = u % sets;
        r.seq = u / sets;
        r.any = r.seq < b.n_seq;
        if (!r.any) return r;
    } else {
        auto begin = [&](int s) { return b.cu_q[s] / TW + int64_t(2) * s; };
        r.seq = last_at_most(b.n_seq, u, begin);
        set = static_cast<int>(u - begin(r.seq));
        r.any = set >= 0;
        if (!r.any) return r;
    }
    r.q = kv_seq(b, r.seq, c.shift);
    r.any = r.q.q > 0;
    if (!r.any) return r;
    r.lo = max(r.q.n - r.q.q, 0);
    r.first = r.lo / kKvGroup * kKvGroup + set * TW;
    r.any = r.first < r.q.n || !r.q.ok;
    return r;
}

// The groups of a run: where their codes begin and which of their tokens are to
// be moved.
template <int TW>
struct Groups {
    uint8_t* block[TW / 16];  // the page's block of the head, null: no such page
    int slot[TW / 16];        // of the group's first token in its page
    uint32_t live;            // a bit for each token of the run

    // ok: the sequence's positions below n are all in the table.
    __device__ Groups(const KvCache& c, const KvBatch& b, const Unit& u) : live(0) {
#pragma unroll
        for (int g = 0; g < TW / 16; g++) {
            const int j = u.first + g * 16;
            const int page = j < u.q.n ? kv_page(b, c, u.seq, j) : -1;
            block[g] = page < 0 ? nullptr : kv_block(c, page, u.head);
            slot[g] = j & ((1 << c.shift) - 1);
            const int from = min(max(u.lo - j, 0), 16), to = min(max(u.q.n - j, 0), 16);
            if (from < to) live |= (((1u << to) - 1) & ~((1u << from) - 1)) << (g * 16);
        }
    }
    __device__ uint32_t held() const {
        uint32_t m = 0;
#pragma unroll
        for (int g = 0; g < TW / 16; g++)
            if (block[g]) m |= 0xffffu << (g * 16);
        return m;
    }
};

// rne(top x / a) in the low bits, half to even.  x * top is exact for 16-bit x and
// the quotient, corrected once by its remainder, is within one unit of 2^-24: a
// quotient half way between codes comes out exactly (it is representable and
// the remainder is exact), and any other is further from half way than that, both
// sides of the comparison being 19-bit integers in one unit.
template <int BITS>
__device__ inline uint32_t code_of(float x, float topf, float a, float inv) {
    const float y = x * topf;
    const float q0 = y * inv;
    const float q = fmaf(fmaf(-q0, a, y), inv, q0);
    // 1.5 * 2^23 rounds at the last bit
    return __float_as_uint(q + (12582912.0f + (BITS == 8 ? 128.0f : 8.0f)));
}

__device__ inline uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400) | __builtin_amdgcn_perm(d, c, 0x0c0c0400) << 16;
}

// A lane's 8 elements from element 8 col of the row at `row` turned to position pos, as rotary.hip
// turns them; f: their frequencies.  In halves the pairs' other elements are another lane's: they are
// read once more, from the cache.
template <int DT, bool VEC>
__device__ inline void turn8(const Rotary& r, const void* base, int64_t row, int col, int64_t pos,
                             const uint64_t* f, float* x) {
    const int el = col * 8, half = r.rot / 2;
    if (el >= r.rot) return;
    if (r.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            if (el + e >= r.rot) break;
            float c, s;
            turn_of(f[e], pos, c, s);
            c *= r.amp, s *= r.sign;
            const float x0 = x[e], x1 = x[e + 1];
            x[e] = fmaf(x0, c, -(x1 * s));
            x[e + 1] = fmaf(x1, c, x0 * s);
        }
        return;
    }
    float y[8];
    if (half % 8 == 0) {
        load8<DT, VEC>(base, row + (el < half ? el + half : el - half), y);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (el + e < r.rot)
                y[e] = load1<DT>(base, row + (el + e < half ? el + e + half : el + e - half));
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (el + e >= r.rot) break;
        float c, s;
        turn_of(f[e], pos, c, s);
        c *= r.amp, s *= r.sign;
        x[e] = fmaf(x[e], c, el + e < half ? -(y[e] * s) : y[e] * s);
    }
}

// HBM-bound: reads 2 T H D elements, writes half (8 bits) or a quarter of that
// in 16-bit types.  A large copy moves 4.8 TB/s; 19192 tokens, 8 heads of 128, 8 bits: 119 MB in
// 31.6 us, 3.8 TB/s, from float32 198 MB in 41.0, 4.8; 4 bits, 8 heads of 64, 16384 tokens 3.1 TB/s and
// 65536 4.1; 64 single tokens 5.1 us.
// ROT: keys are turned to their positions first, in float32, and not rounded before they are held: 48 single
// tokens of 4 heads of 256 6.5 us (8.7 with every row of their runs made into codes).  Over prompts the angles
// bound it, which a lane computes for its 8 elements of each token and head: 4096 tokens, 8 heads of
// 128, 8 bits 14.6 us (9.3 without), 19192 48.1 (30.8), side by side, which has half as many, 38.9.
template <int BITS, int D, int DT, bool VEC, bool SEARCH, bool ROT>
__global__ __launch_bounds__(64 * kWaves) void kv_write_kernel(KvCache c, KvBatch b, KvRows kr,
                                                               KvRows vr, int sets, Rotary rot) {
    using R = Run<BITS, D>;
    __shared__ __align__(16) uint8_t lds[kWaves][R::LDS];
    __shared__ int mags[kWaves][R::TW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane % R::CL, sub = lane / R::CL;
    uint64_t freq[8];
    if constexpr (ROT) {  // first, on their way while the rows are found
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int el = col * 8 + e, half = rot.rot / 2;
            freq[e] = el >= rot.rot ? 0
                                    : rot.turns[rot.interleaved ? el >> 1 : el < half ? el : el - half];
        }
    }
    const Unit u = unit_of<R::TW, SEARCH>(c, b, sets);
    if (!u.any || !u.q.ok) return;  // wave-uniform; the waves share nothing
    const Groups<R::TW> gr(c, b, u);
    const uint32_t live = gr.live & gr.held();
    if (!live) return;
    const KvRows src = u.value ? vr : kr;
    const int64_t row0 = u.q.row + (u.first - (u.q.n - u.q.q));
    float x[R::NI][8];
#pragma unroll
    for (int i = 0; i < R::NI; i++) {
        const int t = i * R::RI + sub;
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
        if (live >> t & 1)
            load8<DT, VEC>(src.p, (row0 + t) * src.tok + u.head * src.head + col * 8, x[i]);
    }
    if constexpr (ROT) {
        if (!u.value) {
#pragma unroll
            for (int i = 0; i < R::NI; i++) {
                const int t = i * R::RI + sub;
                if (live >> t & 1)
                    turn8<DT, VEC>(rot, src.p, (row0 + t) * src.tok + u.head * src.head, col, u.first + t,
                                   freq, x[i]);
            }
        }
    }
    constexpr float top = BITS == 8 ? 127.0f : 7.0f;
#pragma unroll
    for (int i = 0; i < R::NI; i++) {
        // single tokens are one row of a run
        if (ROT && !(live >> (i * R::RI) & ((1u << R::RI) - 1))) continue;
        // |x| as an integer: infinities and NaN are the largest
        int mag = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) mag = max(mag, __float_as_int(x[i][e]) & 0x7fffffff);
#pragma unroll
        for (int o = 1; o < R::CL; o <<= 1) mag = max(mag, __shfl_xor(mag, o));
        const float amax = __int_as_float(mag);
        const bool finite = mag < 0x7f800000, held = finite && amax >= kFloor;
        // top * x must not overflow: very large rows are scaled by 2^-64 first
        const float f = amax > 0x1p100f ? 0x1p-64f : 1.0f;
        const float a = held ? amax * f : 1.0f, topf = held ? top * f : 0.0f;
        const float inv = __builtin_amdgcn_rcpf(a);
        uint32_t d[8];
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] = code_of<BITS>(x[i][e], topf, a, inv);
        u32x2 w = {bytes4(d[0], d[1], d[2], d[3]), bytes4(d[4], d[5], d[6], d[7])};
        if (!finite) w = BITS == 8 ? u32x2{0x80808080u, 0x80808080u} : u32x2{0x08080808u, 0x08080808u};
        const int t = i * R::RI + sub;
        uint8_t* const at = lds[wave] + (t >> 4) * R::NP * kTilePitch + (t & 15) * 16;
        if constexpr (BITS == 8) {
            *reinterpret_cast<u32x2*>(at + (col >> 1) * kTilePitch + (col & 1) * 8) = w;
        } else {
            // the lane D/16 on holds the elements of the high nibbles
            const uint32_t m = 0x0f0f0f0fu;
            const uint32_t h0 = __shfl_xor(static_cast<int>(w[0]), R::CL / 2) & m;
            const uint32_t h1 = __shfl_xor(static_cast<int>(w[1]), R::CL / 2) & m;
            if (col < R::CL / 2)
                *reinterpret_cast<u32x2*>(at + (col >> 1) * kTilePitch + (col & 1) * 8) =
                    u32x2{(w[0] & m) | h0 << 4, (w[1] & m) | h1 << 4};
        }
        if (col == 0) mags[wave][t] = mag;
    }
    wave_lds_fence();
    if (lane < R::TW && (live >> lane & 1)) {
        const float amax = __int_as_float(mags[wave][lane]);
        const float scale = !(amax < INFINITY) ? nan32() : amax >= kFloor ? amax / top : 0.0f;
        const int g = lane >> 4;
        float* const sc = reinterpret_cast<float*>((R::TW == 32 && g ? gr.block[R::TW / 16 - 1] : gr.block[0]) +
                                                   2 * c.codes);
        sc[(u.value << c.shift) + (R::TW == 32 && g ? gr.slot[R::TW / 16 - 1] : gr.slot[0]) +
           (lane & 15)] = scale;
    }
#pragma unroll
    for (int i = 0; i < R::OUT; i++) {
        const int k = lane + 64 * i, g = R::TW == 32 ? k / R::ROW : 0, in = k - g * R::ROW;
        uint8_t* const blk = R::TW == 32 && g ? gr.block[R::TW / 16 - 1] : gr.block[0];
        const int slot = R::TW == 32 && g ? gr.slot[R::TW / 16 - 1] : gr.slot[0];
        const uint32_t mine = live >> (g * 16) & 0xffff;
        if (!u.value) {
            const int t = in / (R::NP * 4) * 4 + (in & 3), piece = in % (R::NP * 4) >> 2;
            const u32x4 w = *reinterpret_cast<const u32x4*>(
                lds[wave] + (g * R::NP + piece) * kTilePitch + t * 16);
            if (mine >> t & 1) *reinterpret_cast<u32x4*>(blk + slot * R::ROW + in * 16) = w;
        } else {
            uint8_t* const tile = lds[wave] + (k >> 4) * kTilePitch;
            transpose16(tile, lane);
            const u32x4 w = *reinterpret_cast<const u32x4*>(tile + (k & 15) * 16);
            uint8_t* const dst = blk + c.codes + slot * R::ROW + in * 16;
            if (mine == 0xffff) {
                *reinterpret_cast<u32x4*>(dst) = w;
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (mine >> r & 1) dst[r] = static_cast<uint8_t>(w[r >> 2] >> (8 * (r & 3)));
            }
        }
    }
}

// HBM-bound: the reverse of kv_write_kernel, out rows contiguous.  316386 tokens, 8 heads
// of 64, 4 bits to float16: 830 MB in 165 us, 5.0 TB/s; elements one by one, as the codes lie, took
// 268 with the write before it, which is now 181 with it.  19192 tokens, 8 heads of 128, 8 bits to
// bfloat16 20.8 us, 5.7 TB/s, to float32 47.4, 4.2.
template <int BITS, int D, int DT, bool VEC, bool SEARCH>
__global__ __launch_bounds__(64 * kWaves) void kv_read_kernel(KvCache c, KvBatch b, void* ko,
                                                              void* vo, int sets) {
    using R = Run<BITS, D>;
    __shared__ __align__(16) uint8_t lds[kWaves][R::LDS];
    __shared__ float scales[kWaves][R::TW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Unit u = unit_of<R::TW, SEARCH>(c, b, sets);
    void* const out = u.value ? vo : ko;
    if (!u.any || !out) return;  // wave-uniform; the waves share nothing
    const Groups<R::TW> gr(c, b, u);
    int64_t row0 = u.q.row + (u.first - (u.q.n - u.q.q));
    uint32_t live = gr.live;
    if (!u.q.ok) {  // no positions to go by: the run's share of the rows becomes NaN
        row0 = u.q.row + u.first;
        live = 0;
        for (int t = 0; t < R::TW; t++)
            if (u.first + t < u.q.q) live |= 1u << t;
    }
    if (lane < R::TW) {
        const int g = lane >> 4;
        const uint8_t* const blk = R::TW == 32 && g ? gr.block[R::TW / 16 - 1] : gr.block[0];
        const int slot = (R::TW == 32 && g ? gr.slot[R::TW / 16 - 1] : gr.slot[0]) + (lane & 15);
        float s = nan32();
        if (blk && (live >> lane & 1))
            s = reinterpret_cast<const float*>(blk + 2 * c.codes)[(u.value << c.shift) + slot];
        scales[wave][lane] = s;
    }
    u32x4 w[R::OUT];
#pragma unroll
    for (int i = 0; i < R::OUT; i++) {
        const int k = lane + 64 * i, g = R::TW == 32 ? k / R::ROW : 0, in = k - g * R::ROW;
        const uint8_t* const blk = R::TW == 32 && g ? gr.block[R::TW / 16 - 1] : gr.block[0];
        const int slot = R::TW == 32 && g ? gr.slot[R::TW / 16 - 1] : gr.slot[0];
        w[i] = u32x4{0, 0, 0, 0};
        if (blk)
            w[i] = *reinterpret_cast<const u32x4*>(blk + (u.value ? c.codes : 0) + slot * R::ROW +
                                                   in * 16);
    }
#pragma unroll
    for (int i = 0; i < R::OUT; i++) {
        const int k = lane + 64 * i, g = R::TW == 32 ? k / R::ROW : 0, in = k - g * R::ROW;
        if (!u.value) {
            const int t = in / (R::NP * 4) * 4 + (in & 3), piece = in % (R::NP * 4) >> 2;
            *reinterpret_cast<u32x4*>(lds[wave] + (g * R::NP + piece) * kTilePitch + t * 16) = w[i];
        } else {
            uint8_t* const tile = lds[wave] + (k >> 4) * kTilePitch;
            *reinterpret_cast<u32x4*>(tile + (k & 15) * 16) = w[i];
            wave_lds_fence();
            transpose16(tile, lane);
        }
    }
    wave_lds_fence();
    const int col = lane % R::CL, sub = lane / R::CL;
    constexpr int HALF = BITS == 8 ? R::CL : R::CL / 2;  // lanes of the low nibbles
    const int byte = col % HALF;
#pragma unroll
    for (int i = 0; i < R::NI; i++) {
        const int t = i * R::RI + sub;
        u32x2 v = *reinterpret_cast<const u32x2*>(lds[wave] +
                                                  ((t >> 4) * R::NP + (byte >> 1)) * kTilePitch +
                                                  (t & 15) * 16 + (byte & 1) * 8);
        if (BITS == 4 && col >= HALF) v >>= 4;
        const float scale = scales[wave][t];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t by = v[e >> 2] >> (8 * (e & 3)) & (BITS == 8 ? 255u : 15u);
            x[e] = (static_cast<float>(by) - (BITS == 8 ? 128.0f : 8.0f)) * scale;
        }
        if (live >> t & 1)
            store8<DT, VEC>(out, ((row0 + t) * c.H + u.head) * D + col * 8, x);
    }
}

// Whole pages, 16 bytes a lane and kCopyDeep of them in flight; HBM-bound: 63 pages of 135 kB, 17 MB, in 5.5 us.
// A pair that names a page that the cache does not have is left out.
constexpr int kCopyDeep = 4;
constexpr int kCopyRun = 256 * 16 * kCopyDeep;  // bytes of a workgroup

__global__ __launch_bounds__(256) void kv_copy_pages_kernel(KvCache c, const int32_t* src,
                                                            const int32_t* dst, int per) {
    const uint32_t pair = blockIdx.x / per, part = blockIdx.x % per;
    const int from = src[pair], to = dst[pair];
    if (from < 0 || from >= c.num_pages || to < 0 || to >= c.num_pages || from == to) return;
    const int64_t bytes = c.block * c.H, at = static_cast<int64_t>(part) * kCopyRun + threadIdx.x * 16;
    const uint8_t* const a = c.base + from * bytes;
    uint8_t* const b = c.base + to * bytes;
    u32x4 v[kCopyDeep];
#pragma unroll
    for (int i = 0; i < kCopyDeep; i++)
        if (at + i * 4096 < bytes) v[i] = *reinterpret_cast<const u32x4*>(a + at + i * 4096);
#pragma unroll
    for (int i = 0; i < kCopyDeep; i++)
        if (at + i * 4096 < bytes) *reinterpret_cast<u32x4*>(b + at + i * 4096) = v[i];
}

// Tokens as they are held, from any slots (page * page_size + place) of cache f to the batch's new
// tokens; latency bounds it: of a head at a time, its loads, then its stores, with three quarters of the
// waves' time spent waiting.  A wave has a run's keys or values in `per` heads: where its tokens lie is the
// same for each.  Keys move 16 bytes a lane, a piece of a token, to where they lie in order.  Values stand
// token by token within a group of 16: a lane makes the 16 bytes of an element from its 16 bytes in
// each of the groups that the tokens come from, kMoveDeep of which are on their way at once (half of
// the tokens at random: three on average).  A slot that the cache does not have counts as a row that
// is not finite.  31187 of 62000 tokens at random, 8 heads of 128, 8 bits: 132 MB in 55 us, 2.4 TB/s (47 where
// calls follow each other; lines of which a part is another token's: 80 MB read for 66, 3 us of a copy);
// 213600 in runs, 8 of 64, 4 bits, 246 MB in 85, 2.9 TB/s (76); 700 tokens 6.4.
constexpr int kMoveDeep = 4;
// Waves that a call is cut into by heads at most: the first of these 51.4 us with 8192, 47.1 with 16384, 49.1
// with one head each; the second 71.2, 75.7, 74.8.
constexpr int kMoveWaves = 16384;

template <int BITS, int D, bool SEARCH>
__global__ __launch_bounds__(64 * kWaves) void kv_copy_kernel(KvCache f, KvCache c, KvBatch b,
                                                              const int64_t* slots, int sets, int per) {
    using R = Run<BITS, D>;
    constexpr uint32_t zero = BITS == 8 ? 0x80808080u : 0x88888888u;  // codes 0
    constexpr int TW = R::TW, NG = TW / 16;
    const int lane = threadIdx.x & 63;
    KvCache parts = c;
    parts.H = (c.H + per - 1) / per;
    const Unit u = unit_of<TW, SEARCH>(parts, b, sets);
    if (!u.any || !u.q.ok) return;  // wave-uniform; the waves share nothing
    const int h0 = u.head * per, h1 = min(h0 + per, c.H);
    // where the run's tokens go: blocks of head 0 (null: no such page), places in them
    uint8_t* dst[NG];
    int to[NG];
    uint32_t live = 0;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const int j = u.first + g * 16;
        const int page = j < u.q.n ? kv_page(b, c, u.seq, j) : -1;
        dst[g] = page < 0 ? nullptr : kv_block(c, page, 0);
        to[g] = j & ((1 << c.shift) - 1);
        const int lo = min(max(u.lo - j, 0), 16), hi = min(max(u.q.n - j, 0), 16);
        if (page >= 0 && lo < hi) live |= (((1u << hi) - 1) & ~((1u << lo) - 1)) << (g * 16);
    }
    if (!live) return;
    // and come from: a token a lane, page -1: none
    const bool mine = lane < TW && (live >> (lane & (TW - 1)) & 1);
    int64_t slot = -1;
    if (mine) slot = slots[u.q.row + (u.first - (u.q.n - u.q.q)) + lane];
    if (slot < 0 || slot >> f.shift >= f.num_pages) slot = -1;
    const int page = slot < 0 ? -1 : static_cast<int>(slot >> f.shift);
    const int place = static_cast<int>(slot) & ((1 << f.shift) - 1);
    auto block = [&](int g) { return NG == 2 && g ? dst[NG - 1] : dst[0]; };
    auto place_of = [&](int g) { return NG == 2 && g ? to[NG - 1] : to[0]; };
    auto scale = [&](int h) {
        if (!mine) return;
        float s = nan32();
        if (page >= 0)
            s = reinterpret_cast<const float*>(kv_block(f, page, h) + 2 * f.codes)[(u.value << f.shift) + place];
        reinterpret_cast<float*>(block(lane >> 4) + h * c.block + 2 * c.codes)[
            (u.value << c.shift) + place_of(lane >> 4) + (lane & 15)] = s;
    };
    if (!u.value) {
        const uint8_t* from[R::OUT];
        int64_t at[R::OUT];
        bool has[R::OUT];
#pragma unroll
        for (int i = 0; i < R::OUT; i++) {
            const int k = lane + 64 * i, g = TW == 32 ? k / R::ROW : 0, in = k - g * R::ROW;
            const int t = in / (R::NP * 4) * 4 + (in & 3), piece = in % (R::NP * 4) >> 2;
            const int pg = __shfl(page, g * 16 + t), pl = __shfl(place, g * 16 + t);
            from[i] = pg < 0 ? nullptr
                             : kv_block(f, pg, 0) + (pl & ~3) * R::ROW + piece * 64 + (pl & 3) * 16;
            has[i] = live >> (g * 16 + t) & 1;
            at[i] = has[i] ? block(g) - c.base + place_of(g) * R::ROW + in * 16 : 0;
        }
        for (int h = h0; h < h1; h++) {
            u32x4 w[R::OUT];
#pragma unroll
            for (int i = 0; i < R::OUT; i++) {
                w[i] = u32x4{zero, zero, zero, zero};
                if (from[i]) w[i] = *reinterpret_cast<const u32x4*>(from[i] + h * f.block);
            }
            scale(h);
#pragma unroll
            for (int i = 0; i < R::OUT; i++)
                if (has[i]) *reinterpret_cast<u32x4*>(c.base + at[i] + h * c.block) = w[i];
        }
        return;
    }
    // Byte columns of a lane; rows of fewer than 64 bytes: two heads at once.
    constexpr int COLS = (R::ROW + 63) / 64, HP = R::ROW < 64 ? 64 / R::ROW : 1;
    const int col = lane % (R::ROW < 64 ? R::ROW : 64), sub = lane / (R::ROW < 64 ? R::ROW : 64);
    // the tokens whose group is another than the token's before
    uint32_t first[NG];
    const int group = place & ~15;
    const int pg0 = __shfl(page, max(lane - 1, 0)), gp0 = __shfl(group, max(lane - 1, 0));
    const uint64_t differ = __ballot(page != pg0 || group != gp0);
#pragma unroll
    for (int g = 0; g < NG; g++) first[g] = (differ >> (g * 16) & 0xffff) | 1;
    for (int hb = h0; hb < h1; hb += HP) {
        const int h = min(hb + sub, h1 - 1);
        const bool here = hb + sub < h1;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const uint32_t part = live >> (g * 16) & 0xffff;
            if (!part) continue;
            u32x4 out[COLS];
#pragma unroll
            for (int i = 0; i < COLS; i++) out[i] = u32x4{0, 0, 0, 0};
            uint32_t left = first[g];
            while (left) {
                u32x4 v[kMoveDeep][COLS];
                uint32_t tokens[kMoveDeep];
#pragma unroll
                for (int k = 0; k < kMoveDeep; k++) {
                    tokens[k] = 0;
                    if (!left) continue;
                    const uint32_t low = left & -left;
                    left ^= low;
                    // from this first token to before the next
                    tokens[k] = (left ? (left & -left) : 0x10000u) - low;
                    const int t = g * 16 + __builtin_ctz(low);
                    const int p = __builtin_amdgcn_readlane(page, t), at = __builtin_amdgcn_readlane(group, t);
#pragma unroll
                    for (int i = 0; i < COLS; i++) {
                        v[k][i] = u32x4{zero, zero, zero, zero};
                        if (p >= 0)
                            v[k][i] = *reinterpret_cast<const u32x4*>(kv_block(f, p, h) + f.codes + at * R::ROW +
                                                                      (col + 64 * i) * 16);
                    }
                }
#pragma unroll
                for (int k = 0; k < kMoveDeep; k++) {
                    if (!tokens[k]) continue;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        if (!(tokens[k] >> r & 1)) continue;
                        const uint32_t x = __builtin_amdgcn_readlane(place, g * 16 + r) & 15;
                        // byte x of 16 to byte r % 4 of a word: 0x0c makes a zero
                        const uint32_t keep = 0x0c0c0c0cu & ~(0xffu << (8 * (r & 3)));
                        const uint32_t lo = keep | (x < 8 ? x : 0x0c) << (8 * (r & 3));
                        const uint32_t hi = keep | (x < 8 ? 0x0c : x - 8) << (8 * (r & 3));
#pragma unroll
                        for (int i = 0; i < COLS; i++)
                            out[i][r >> 2] |= __builtin_amdgcn_perm(v[k][i][1], v[k][i][0], lo) |
                                              __builtin_amdgcn_perm(v[k][i][3], v[k][i][2], hi);
                    }
                }
            }
            uint8_t* const into = block(g) + h * c.block + c.codes + place_of(g) * R::ROW;
#pragma unroll
            for (int i = 0; i < COLS; i++) {
                uint8_t* const x = into + (col + 64 * i) * 16;
                if (!here) continue;
                if (part == 0xffff) {
                    *reinterpret_cast<u32x4*>(x) = out[i];
                } else {
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (part >> r & 1) x[r] = static_cast<uint8_t>(out[i][r >> 2] >> (8 * (r & 3)));
                }
            }
        }
#pragma unroll
        for (int k = 0; k < HP; k++)
            if (hb + k < h1) scale(hb + k);
    }
}

// The launch's units: every head, keys and values, of each sequence's runs of max_q tokens
// (one more than they fill, for a run that starts inside a group), or of the runs that n_tokens
// tokens can have in n_seq sequences (sets 0) where those are fewer by a third: 5509 tokens of 3
// sequences in and out, a head of 256, 561 and 350 runs: 15.0 us without a search, 13.8 with; 303 of
// 3, 8 heads of 256, 33 and 24 runs: 12.1, 12.7.  False where they do not fit a launch.
bool units(const KvBatch& b, const KvCache& c, int TW, int* sets, unsigned* blocks) {
    const int64_t each = (static_cast<int64_t>(b.max_q) + 15 + TW - 1) / TW;
    const int64_t all = b.n_tokens / TW + int64_t(2) * b.n_seq;
    const bool search = 2 * each * b.n_seq > 3 * all;
    const int64_t runs = search ? all : each * b.n_seq;
    *sets = search ? 0 : static_cast<int>(each);
    if (runs >= int64_t(1) << 31) return false;
    const int64_t n = (runs * c.H * 2 + kWaves - 1) / kWaves;
    *blocks = static_cast<unsigned>(n);
    return n < int64_t(1) << 23;
}

// f<BITS, D, DT, VEC> for the run-time values.
template <template <int, int, int, bool> class F, typename... A>
hipError_t pick(int bits, int D, int dt, bool vec, A&&... a) {
#define JHQ_KV_V(B, DD, T) return vec ? F<B, DD, T, true>::run(a...) : F<B, DD, T, false>::run(a...)
#define JHQ_KV_T(B, DD)                              \
    switch (dt) {                                    \
        case JHQ_F32: JHQ_KV_V(B, DD, JHQ_F32);      \
        case JHQ_BF16: JHQ_KV_V(B, DD, JHQ_BF16);    \
        default: JHQ_KV_V(B, DD, JHQ_F16);           \
    }
#define JHQ_KV_D(B)                    \
    switch (D) {                       \
        case 64: JHQ_KV_T(B, 64)       \
        case 128: JHQ_KV_T(B, 128)     \
        default: JHQ_KV_T(B, 256)      \
    }
    if (bits == 8) JHQ_KV_D(8) else JHQ_KV_D(4)
#undef JHQ_KV_D
#undef JHQ_KV_T
#undef JHQ_KV_V
}

template <int BITS, int D, int DT, bool VEC>
struct Write {
    static hipError_t run(const KvCache& c, const KvBatch& b, const KvRows& k, const KvRows& v,
                          const Rotary* r, hipStream_t s) {
        int sets;
        unsigned blocks;
        if (!units(b, c, Run<BITS, D>::TW, &sets, &blocks)) return hipErrorInvalidValue;
        auto go = [&](auto kernel) {
            kernel<<<blocks, 64 * kWaves, 0, s>>>(c, b, k, v, sets, r ? *r : Rotary{});
            return hipGetLastError();
        };
        if (r)
            return sets ? go(kv_write_kernel<BITS, D, DT, VEC, false, true>)
                        : go(kv_write_kernel<BITS, D, DT, VEC, true, true>);
        return sets ? go(kv_write_kernel<BITS, D, DT, VEC, false, false>)
                    : go(kv_write_kernel<BITS, D, DT, VEC, true, false>);
    }
};

template <int BITS, int D, int DT, bool VEC>
struct Read {
    static hipError_t run(const KvCache& c, const KvBatch& b, void* k, void* v, hipStream_t s) {
        int sets;
        unsigned blocks;
        if (!units(b, c, Run<BITS, D>::TW, &sets, &blocks)) return hipErrorInvalidValue;
        if (sets)
            kv_read_kernel<BITS, D, DT, VEC, false><<<blocks, 64 * kWaves, 0, s>>>(c, b, k, v, sets);
        else
            kv_read_kernel<BITS, D, DT, VEC, true><<<blocks, 64 * kWaves, 0, s>>>(c, b, k, v, sets);
        return hipGetLastError();
    }
};

template <int BITS, int D>
hipError_t copy_run(const KvCache& f, const KvCache& c, const KvBatch& b, const int64_t* slots,
                    hipStream_t s) {
    constexpr int TW = Run<BITS, D>::TW, HP = Run<BITS, D>::ROW < 64 ? 64 / Run<BITS, D>::ROW : 1;
    int sets;
    unsigned blocks;
    // a wave has as many heads as leave enough waves for the chip
    KvCache parts = c;
    parts.H = 1;
    if (!units(b, parts, TW, &sets, &blocks)) return hipErrorInvalidValue;
    const int64_t waves = static_cast<int64_t>(blocks) * kWaves;
    const int64_t most = waves * c.H / kMoveWaves;
    const int per = static_cast<int>(std::min<int64_t>(c.H, std::max<int64_t>(HP, most / HP * HP)));
    parts.H = (c.H + per - 1) / per;
    if (!units(b, parts, TW, &sets, &blocks)) return hipErrorInvalidValue;
    if (sets)
        kv_copy_kernel<BITS, D, false><<<blocks, 64 * kWaves, 0, s>>>(f, c, b, slots, sets, per);
    else
        kv_copy_kernel<BITS, D, true><<<blocks, 64 * kWaves, 0, s>>>(f, c, b, slots, sets, per);
    return hipGetLastError();
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

hipError_t kv_write(const KvCache& c, const KvBatch& b, int bits, int D, const KvRows& k,
                    const KvRows& v, int dtype, const Rotary* r, hipStream_t s) {
    // 16-byte loads where every row starts on 16 bytes
    const int e = dtype == JHQ_F32 ? 4 : 8;
    const bool vec = aligned16(k.p) && aligned16(v.p) && k.tok % e == 0 && k.head % e == 0 &&
                     v.tok % e == 0 && v.head % e == 0;
    return pick<Write>(bits, D, dtype, vec, c, b, k, v, r, s);
}

hipError_t kv_read(const KvCache& c, const KvBatch& b, int bits, int D, void* k, void* v, int dtype,
                   hipStream_t s) {
    return pick<Read>(bits, D, dtype, aligned16(k) && aligned16(v), c, b, k, v, s);
}

hipError_t kv_copy(const KvCache& f, const KvCache& c, const KvBatch& b, int bits, int D,
                   const int64_t* slots, hipStream_t s) {
    if (bits == 8)
        return D == 64    ? copy_run<8, 64>(f, c, b, slots, s)
               : D == 128 ? copy_run<8, 128>(f, c, b, slots, s)
                          : copy_run<8, 256>(f, c, b, slots, s);
    return D == 64    ? copy_run<4, 64>(f, c, b, slots, s)
           : D == 128 ? copy_run<4, 128>(f, c, b, slots, s)
                      : copy_run<4, 256>(f, c, b, slots, s);
}

hipError_t kv_copy_pages(const KvCache& c, const int32_t* src, const int32_t* dst, int64_t n,
                         hipStream_t s) {
    const int64_t per = (c.block * c.H + kCopyRun - 1) / kCopyRun;
    if (n >= 1 << 23 || n * per >= 1 << 23) return hipErrorInvalidValue;
    kv_copy_pages_kernel<<<static_cast<unsigned>(n * per), 256, 0, s>>>(c, src, dst,
                                                                       static_cast<int>(per));
    return hipGetLastError();
}

}  // namespace jhq

// ---------------------------------------------------------------------------
// C-ABI
// ---------------------------------------------------------------------------

namespace {

int bad(const std::string& msg) { return jhq_set_error(JHQ_EINVAL, msg.c_str()); }

int launched(const char* what, hipError_t e) {
    if (e == hipSuccess) return JHQ_OK;
    (void)hipGetLastError();  // reported here: not the next launch's
    if (e == hipErrorInvalidValue)
        return bad(std::string(what) + ": more work than one launch holds");
    return jhq_set_error(e == hipErrorOutOfMemory ? JHQ_ENOMEM : JHQ_EDEVICE,
                         (std::string(what) + ": " + hipGetErrorString(e)).c_str());
}

int check_params(const jhq_kv_params* p) {
    if (!p) return bad("null parameters");
    if (p->bits != 8 && p->bits != 4) return bad("bits must be 8 or 4");
    if (p->kv_heads < 1 || p->kv_heads > 1024) return bad("kv_heads must be 1 .. 1024");
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
        return bad("head_dim must be 64, 128 or 256");
    if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
        return bad("page_size must be a power of two, 16 .. 1024");
    if (p->num_pages < 1 || p->num_pages > INT32_MAX) return bad("num_pages must be 1 .. 2^31 - 1");
    return JHQ_OK;
}

// Positions, a window before one, and the steps a kernel goes past the end stay
// within int.  A window as long as the longest sequence is none, so longer ones are cut.
constexpr int kMaxTokens = 1 << 30;

int check_batch(const jhq_kv_batch* b) {
    if (!b) return bad("null batch");
    if (b->n_seq < 0 || b->max_pages < 0 || b->n_tokens < 0 || b->max_q < 0 || b->max_kv < 0)
        return bad("negative size in the batch");
    if (b->max_kv > kMaxTokens || b->max_q > kMaxTokens)
        return bad("max_q and max_kv are at most 2^30");
    if (b->n_seq > 0 && (!b->d_kv_len || !b->d_cu_q || (b->max_pages > 0 && !b->d_pages)))
        return bad("null array in the batch");
    return JHQ_OK;
}

int64_t block_bytes(const jhq_kv_params& p) {
    return static_cast<int64_t>(p.page_size) * (p.head_dim * p.bits / 8 * 2 + 8);
}

jhq::KvCache cache_of(const jhq_kv_params& p, const void* base) {
    jhq::KvCache c;
    c.base = static_cast<uint8_t*>(const_cast<void*>(base));
    c.block = block_bytes(p);
    c.num_pages = static_cast<int32_t>(p.num_pages);
    c.H = p.kv_heads;
    c.shift = __builtin_ctz(static_cast<unsigned>(p.page_size));
    c.codes = p.page_size * p.head_dim * p.bits / 8;
    return c;
}

// cu_q names no row past 2^31 - 1.
jhq::KvBatch batch_of(const jhq_kv_batch& b) {
    const int64_t rows = std::min<int64_t>(b.n_tokens, INT32_MAX);
    return {b.d_pages, b.d_kv_len, b.d_cu_q, rows, b.n_seq, b.max_pages, b.max_q, b.max_kv};
}

int check_cache(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b) {
    int rc = check_params(p);
    if (rc == JHQ_OK) rc = check_batch(b);
    if (rc != JHQ_OK) return rc;
    if (!d_cache) return bad("null cache");
    if (!jhq::aligned16(d_cache)) return bad("the cache must be 16-byte aligned");
    return JHQ_OK;
}

// f's result; an exception (no memory for a message) does not leave a C entry point.
template <class T, class F>
T entry(T failed, F f) noexcept {
    try {
        return f();
    } catch (...) {
        return failed;
    }
}

bool idle(const jhq_kv_batch* b) { return b->n_seq == 0 || b->n_tokens == 0 || b->max_q == 0; }

int check_heads(const jhq_kv_params* p, int q_heads, int window) {
    if (q_heads < 1 || q_heads % p->kv_heads) return bad("q_heads must be a multiple of kv_heads");
    if (q_heads > 16384) return bad("q_heads must be at most 16384");
    if (window < 0) return bad("window must not be negative");
    return JHQ_OK;
}

int64_t do_bytes(const jhq_kv_params* p) {
    if (check_params(p) != JHQ_OK) return 0;
    // at most 2^31 pages x 2^10 heads x 2^10 tokens x 520 bytes: past 2^60
    const __int128 n = static_cast<__int128>(p->num_pages) * p->kv_heads * block_bytes(*p);
    if (n > (int64_t(1) << 50)) {
        bad("the cache would have more than 2^50 bytes");
        return 0;
    }
    return static_cast<int64_t>(n);
}

int do_write(const jhq_kv_params* p, void* d_cache, const jhq_kv_batch* b, const void* d_k,
             int64_t k_tok, int64_t k_head, const void* d_v, int64_t v_tok, int64_t v_head,
             int dtype, const jhq_rotary* r, void* stream) {
    const int rc = check_cache(p, d_cache, b);
    if (rc != JHQ_OK) return rc;
    jhq::Rotary rot = {};
    if (r) {
        const std::string wrong = jhq::rotary_wrong(r);
        if (!wrong.empty()) return bad(wrong);
        if (r->head_dim != p->head_dim) return bad("rotary: head_dim is another than the cache's");
        rot = jhq::rotary_of(*r, false);
    }
    if (dtype != JHQ_F32 && dtype != JHQ_BF16 && dtype != JHQ_F16)
        return bad("keys and values must be JHQ_F32, JHQ_BF16 or JHQ_F16");
    if (idle(b)) return JHQ_OK;
    if (!d_k || !d_v) return bad("null keys or values");
    return launched("kv_write", jhq::kv_write(cache_of(*p, d_cache), batch_of(*b), p->bits,
                                              p->head_dim, {d_k, k_tok, k_head},
                                              {d_v, v_tok, v_head}, dtype, r ? &rot : nullptr,
                                              static_cast<hipStream_t>(stream)));
}

int do_read(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b, void* d_k,
                 void* d_v, int dtype, void* stream) {
    const int rc = check_cache(p, d_cache, b);
    if (rc != JHQ_OK) return rc;
    if (dtype != JHQ_F32 && dtype != JHQ_BF16 && dtype != JHQ_F16)
        return bad("keys and values must be JHQ_F32, JHQ_BF16 or JHQ_F16");
    if (idle(b) || (!d_k && !d_v)) return JHQ_OK;
    return launched("kv_read", jhq::kv_read(cache_of(*p, d_cache), batch_of(*b), p->bits,
                                            p->head_dim, d_k, d_v, dtype,
                                            static_cast<hipStream_t>(stream)));
}

int do_copy_pages(const jhq_kv_params* p, void* d_cache, const int32_t* d_src, const int32_t* d_dst,
                  int64_t n, void* stream) {
    const int rc = check_params(p);
    if (rc != JHQ_OK) return rc;
    if (!d_cache) return bad("null cache");
    if (!jhq::aligned16(d_cache)) return bad("the cache must be 16-byte aligned");
    if (n < 0) return bad("negative number of pages");
    if (n == 0) return JHQ_OK;
    if (!d_src || !d_dst) return bad("null pages");
    return launched("kv_copy_pages", jhq::kv_copy_pages(cache_of(*p, d_cache), d_src, d_dst, n,
                                                        static_cast<hipStream_t>(stream)));
}

int do_copy(const jhq_kv_params* from, const void* d_from, const int64_t* d_slots,
            const jhq_kv_params* p, void* d_cache, const jhq_kv_batch* b, void* stream) {
    int rc = check_cache(p, d_cache, b);
    if (rc == JHQ_OK) rc = check_params(from);
    if (rc != JHQ_OK) return rc;
    if (!d_from) return bad("null source cache");
    if (!jhq::aligned16(d_from)) return bad("the source cache must be 16-byte aligned");
    if (from->bits != p->bits || from->kv_heads != p->kv_heads || from->head_dim != p->head_dim)
        return bad("the source cache has other bits, heads or elements");
    if (idle(b)) return JHQ_OK;
    if (!d_slots) return bad("null slots");
    return launched("kv_copy", jhq::kv_copy(cache_of(*from, d_from), cache_of(*p, d_cache), batch_of(*b),
                                            p->bits, p->head_dim, d_slots,
                                            static_cast<hipStream_t>(stream)));
}

// What attention needs; lead: the sequences' prefixes, or null.  -1 and a message where an argument is
// not valid.
int64_t do_work_bytes(const jhq_kv_params* p, const jhq_kv_batch* b, const jhq_kv_batch* lead, int once,
                      int q_heads, int window) {
    if (check_params(p) != JHQ_OK || check_batch(b) != JHQ_OK ||
        check_heads(p, q_heads, window) != JHQ_OK)
        return -1;
    if (lead) {
        if (check_batch(lead) != JHQ_OK) return -1;
        if (lead->n_tokens != b->n_tokens) {
            bad("the prefix has another number of rows than the batch");
            return -1;
        }
        if (once != 0 && once != 1) {
            bad("once must be 0 or 1");
            return -1;
        }
    }
    if (idle(b)) return 0;
    // rows and positions are ints in the kernels
    const int G = q_heads / p->kv_heads;
    if (static_cast<int64_t>(b->max_q) * G > 1 << 30 || (lead && static_cast<int64_t>(lead->max_q) * G > 1 << 30)) {
        bad("max_q * q_heads / kv_heads must be at most 2^30");
        return -1;
    }
    const jhq::KvCache c = cache_of(*p, nullptr);
    const int64_t n = lead ? jhq::kv_shared_work(c, batch_of(*lead), batch_of(*b), p->head_dim, G, once)
                           : jhq::kv_attend_work(c, batch_of(*b), p->head_dim, G, window);
    if (n < 0) bad("the workspace would have more than 2^50 bytes");
    return n;
}

int do_attend(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b,
              const jhq_kv_batch* lead, int once, const void* d_q, int64_t q_tok, int64_t q_head, int q_heads,
              int dtype, float scale, int causal, int window, void* d_out, float* d_lse, void* d_work,
              int64_t work_bytes, void* stream) {
    int rc = check_cache(p, d_cache, b);
    if (rc == JHQ_OK) rc = check_heads(p, q_heads, window);
    if (rc != JHQ_OK) return rc;
    if (dtype != JHQ_BF16 && dtype != JHQ_F16) return bad("queries must be JHQ_BF16 or JHQ_F16");
    if (causal != 0 && causal != 1) return bad("causal must be 0 or 1");
    if (window && !causal) return bad("a window needs causal = 1");
    if (!std::isfinite(scale)) return bad("scale must be finite");
    const int64_t need = lead || !idle(b) ? do_work_bytes(p, b, lead, once, q_heads, window) : 0;
    if (need < 0) return JHQ_EINVAL;
    if (idle(b)) return JHQ_OK;
    if (!d_q || !d_out) return bad("null queries or output");
    if (need > 0 && !d_work) return bad("null workspace");
    if (work_bytes < need)
        return bad("the workspace has " + std::to_string(work_bytes) + " bytes, " +
                   std::to_string(need) + " are needed (jhq_kv_work_bytes)");
    if (!jhq::aligned16(d_work)) return bad("the workspace must be 16-byte aligned");
    const int q16 = jhq::aligned16(d_q) && q_tok % 8 == 0 && q_head % 8 == 0;
    const int out8 = (reinterpret_cast<uintptr_t>(d_out) & 7) == 0;
    const jhq::KvAttend a = {{d_q, q_tok, q_head}, q_heads, q_heads / p->kv_heads, dtype, scale,
                             causal, std::min(window, kMaxTokens), d_out, q16, out8, d_lse, static_cast<float*>(d_work)};
    const jhq::KvCache c = cache_of(*p, d_cache);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return launched("kv_attend",
                    lead ? jhq::kv_attend_shared(c, batch_of(*lead), batch_of(*b), p->bits, p->head_dim, a, once, s)
                         : jhq::kv_attend(c, batch_of(*b), p->bits, p->head_dim, a, s));
}

}  // namespace

extern "C" {

int64_t jhq_kv_bytes(const jhq_kv_params* p) {
    return entry(int64_t(0), [&] { return do_bytes(p); });
}

int64_t jhq_kv_work_bytes(const jhq_kv_params* p, const jhq_kv_batch* b, int q_heads, int window) {
    return entry(int64_t(-1), [&] { return do_work_bytes(p, b, nullptr, 0, q_heads, window); });
}

int64_t jhq_kv_shared_work_bytes(const jhq_kv_params* p, const jhq_kv_batch* b, const jhq_kv_batch* prefix,
                                 int once, int q_heads) {
    return entry(int64_t(-1), [&]() -> int64_t {
        if (prefix) return do_work_bytes(p, b, prefix, once, q_heads, 0);
        bad("null prefix");
        return -1;
    });
}

int jhq_k_kv_write(const jhq_kv_params* p, void* d_cache, const jhq_kv_batch* b, const void* d_k,
                   int64_t k_tok, int64_t k_head, const void* d_v, int64_t v_tok, int64_t v_head,
                   int dtype, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM), [&] {
        return do_write(p, d_cache, b, d_k, k_tok, k_head, d_v, v_tok, v_head, dtype, nullptr, stream);
    });
}

int jhq_k_kv_write_rotary(const jhq_kv_params* p, void* d_cache, const jhq_kv_batch* b, const void* d_k,
                          int64_t k_tok, int64_t k_head, const void* d_v, int64_t v_tok,
                          int64_t v_head, int dtype, const jhq_rotary* r, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM), [&] {
        if (!r) return bad("null rotary parameters");
        return do_write(p, d_cache, b, d_k, k_tok, k_head, d_v, v_tok, v_head, dtype, r, stream);
    });
}

int jhq_k_kv_read(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b, void* d_k,
                  void* d_v, int dtype, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM), [&] { return do_read(p, d_cache, b, d_k, d_v, dtype, stream); });
}

int jhq_k_kv_copy_pages(const jhq_kv_params* p, void* d_cache, const int32_t* d_src,
                        const int32_t* d_dst, int64_t n, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM),
                 [&] { return do_copy_pages(p, d_cache, d_src, d_dst, n, stream); });
}

int jhq_k_kv_copy(const jhq_kv_params* from, const void* d_from, const int64_t* d_slots,
                  const jhq_kv_params* p, void* d_cache, const jhq_kv_batch* b, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM),
                 [&] { return do_copy(from, d_from, d_slots, p, d_cache, b, stream); });
}

int jhq_k_kv_attend(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b,
                    const void* d_q, int64_t q_tok, int64_t q_head, int q_heads, int dtype,
                    float scale, int causal, int window, void* d_out, float* d_lse, void* d_work,
                    int64_t work_bytes, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM), [&] {
        return do_attend(p, d_cache, b, nullptr, 0, d_q, q_tok, q_head, q_heads, dtype, scale, causal, window,
                         d_out, d_lse, d_work, work_bytes, stream);
    });
}

int jhq_k_kv_attend_shared(const jhq_kv_params* p, const void* d_cache, const jhq_kv_batch* b,
                           const jhq_kv_batch* prefix, int once, const void* d_q, int64_t q_tok, int64_t q_head,
                           int q_heads, int dtype, float scale, int causal, void* d_out, float* d_lse,
                           void* d_work, int64_t work_bytes, void* stream) {
    return entry(static_cast<int>(JHQ_ENOMEM), [&] {
        if (!prefix) return bad("null prefix");
        return do_attend(p, d_cache, b, prefix, once, d_q, q_tok, q_head, q_heads, dtype, scale, causal, 0, d_out,
                         d_lse, d_work, work_bytes, stream);
    });
}

}  // extern "C"
