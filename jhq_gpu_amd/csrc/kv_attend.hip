// kv_attend.hip — attention of new tokens over the quantised key/value cache.
#include "kvcache.h"

#include <hip/hip_runtime.h>

namespace jhq {
namespace {

template <int DT>
__device__ inline float load_el(const void* p, int64_t i) {
    if constexpr (DT == JHQ_BF16)
        return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
    else
        return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}

template <int DT>
__device__ inline void store_el(void* p, int64_t i, float f) {
    if constexpr (DT == JHQ_BF16)
        static_cast<__bf16*>(p)[i] = static_cast<__bf16>(f);
    else
        static_cast<_Float16*>(p)[i] = static_cast<_Float16>(f);
}

// One wave per (row, head): a lane scores one token of 64, then sums the byte
// columns e = lane, lane + 64, ... of the values.
template <int BITS, int D, int DT>
__global__ __launch_bounds__(64) void kv_attend_kernel(KvCache c, KvBatch b, KvAttend a) {
    constexpr int ROW = D * BITS / 8, EC = (ROW + 63) / 64, EL = BITS == 8 ? 1 : 2;
    __shared__ float qs[D], ps[64];
    __shared__ int pg[64];
    const int lane = threadIdx.x, hq = blockIdx.y, seq = blockIdx.z, h = hq / a.G;
    const int Hq = c.H * a.G;
    const KvSeq s = kv_seq(b, seq, c.shift);
    const int i = blockIdx.x;
    if (i >= s.q) return;
    const int64_t row = s.row + i, orow = (row * Hq + hq) * D;
    const int pos = s.n - s.q + i;
    for (int d = lane; d < D; d += 64)
        qs[d] = load_el<DT>(a.q.p, row * a.q.tok + hq * a.q.head + d);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[EC * EL] = {};
    const int hi = s.ok ? (a.causal ? min(pos + 1, s.n) : s.n) : 0;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0;
    for (int j0 = lo & ~63; j0 < hi; j0 += 64) {
        const int j = j0 + lane, slot = j & ((1 << c.shift) - 1);
        const bool see = j >= lo && j < hi;
        const int page = see ? kv_page(b, c, seq, j) : -1;
        const uint8_t* blk = kv_block(c, max(page, 0), h);
        const float* sc = reinterpret_cast<const float*>(blk + 2 * c.codes);
        float ks = 0, vs = 0, dot = 0;
        if (see) ks = vs = NAN;
        if (page >= 0) {
            ks = sc[slot];
            vs = sc[(1 << c.shift) + slot];
            const uint8_t* kp = blk + (slot & ~15) * ROW + (slot & 15) * 16;
            for (int e = 0; e < ROW; e++) {
                const int by = kp[(e >> 4) * 256 + (e & 15)];
                if (BITS == 8)
                    dot = fmaf(qs[e], by - 128.0f, dot);
                else
                    dot = fmaf(qs[e], (by & 15) - 8.0f, fmaf(qs[e + D / 2], (by >> 4) - 8.0f, dot));
            }
        }
        const float x = see ? dot * ks * a.scale : -INFINITY;
        float mt = x;
        for (int k = 1; k < 64; k <<= 1) mt = fmaxf(mt, __shfl_xor(mt, k));
        const float mn = fmaxf(m, mt);
        const float p = see ? expf(x - mn) : 0.0f;
        const float al = mn == -INFINITY ? 1.0f : expf(m - mn);
        float pl = p;
        for (int k = 1; k < 64; k <<= 1) pl += __shfl_xor(pl, k);
        l = l * al + pl;
        m = mn;
        __syncthreads();
        ps[lane] = see ? p * vs : 0.0f;
        pg[lane] = page;
        __syncthreads();
        for (int k = 0; k < EC * EL; k++) o[k] *= al;
        for (int t = 0; t < 64; t++) {
            const int sl = (j0 + t) & ((1 << c.shift) - 1);
            const uint8_t* vb = kv_block(c, max(pg[t], 0), h) + c.codes + (sl & ~15) * ROW + (sl & 15);
            for (int k = 0; k < EC; k++) {
                const int e = lane + k * 64;
                if (e >= ROW) continue;
                const int by = pg[t] >= 0 ? vb[e * 16] : 0;
                if (BITS == 8) {
                    o[k] = fmaf(ps[t], by - 128.0f, o[k]);
                } else {
                    o[2 * k] = fmaf(ps[t], (by & 15) - 8.0f, o[2 * k]);
                    o[2 * k + 1] = fmaf(ps[t], (by >> 4) - 8.0f, o[2 * k + 1]);
                }
            }
        }
    }
    const float r = s.ok ? (l == 0.0f ? 0.0f : 1.0f / l) : NAN;
    for (int k = 0; k < EC; k++) {
        const int e = lane + k * 64;
        if (e >= ROW) continue;
        store_el<DT>(a.out, orow + e, o[k * EL] * r);
        if (BITS == 4) store_el<DT>(a.out, orow + e + D / 2, o[2 * k + 1] * r);
    }
    if (a.lse && lane == 0)
        a.lse[row * Hq + hq] = s.ok ? (l == 0.0f ? -INFINITY : m + logf(l)) : NAN;
}

}  // namespace

int64_t kv_attend_work(const KvCache&, const KvBatch&, int, int, int) { return 0; }

hipError_t kv_attend(const KvCache& c, const KvBatch& b, int bits, int D, const KvAttend& a,
                     int dtype, hipStream_t s) {
    if (c.H * a.G > 65535 || b.n_seq > 65535) return hipErrorInvalidValue;
    const dim3 grid(b.max_q, c.H * a.G, b.n_seq);
#define JHQ_GO(B, DD)                                                        \
    if (dtype == JHQ_BF16)                                                   \
        kv_attend_kernel<B, DD, JHQ_BF16><<<grid, 64, 0, s>>>(c, b, a);      \
    else                                                                     \
        kv_attend_kernel<B, DD, JHQ_F16><<<grid, 64, 0, s>>>(c, b, a)
    if (bits == 8) {
        if (D == 64) { JHQ_GO(8, 64); } else if (D == 128) { JHQ_GO(8, 128); } else { JHQ_GO(8, 256); }
    } else {
        if (D == 64) { JHQ_GO(4, 64); } else if (D == 128) { JHQ_GO(4, 128); } else { JHQ_GO(4, 256); }
    }
#undef JHQ_GO
    return hipGetLastError();
}

}  // namespace jhq
