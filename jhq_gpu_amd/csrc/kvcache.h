// kvcache.h — the quantised key/value cache: its layout in memory and the
// launchers of its kernels.  Internal to kvcache.hip and kv_attend.hip.
#pragma once
#include "../../include/jhq.h"

#include <hip/hip_runtime.h>
#include <cstdint>

namespace jhq {

// Tokens of a code group: pages are whole groups, and a group's keys and
// values are each one contiguous run of 16 * row_bytes bytes.
constexpr int kKvGroup = 16;

// The cache as kernels see it.  Block (page, head) starts at
// base + (page * H + head) * block; in it
//   [0, codes)            key codes, 4 tokens after 4 tokens: piece p of token t: the
//                         16 bytes at (t / 4) * 4 * row + p * 64 + (t % 4) * 16
//   [codes, 2 codes)      value codes, 16 tokens after 16 tokens: byte column e of
//                         token t: the byte at (t / 16) * 16 * row + e * 16 + t % 16
//   then page_size key scales and page_size value scales (float)
// with row = D * bits / 8 bytes per token.  A code is stored unsigned, c + 128
// in 8 bits and c + 8 in 4.  Byte e of a row holds element e in 8 bits, and
// elements e (low nibble) and e + D/2 (high) in 4.
struct KvCache {
    uint8_t* base;
    int64_t block;     // bytes of a (page, head) block
    int32_t num_pages;
    int H, shift;      // page_size = 1 << shift
    int codes;         // bytes of a block's key codes
};

struct KvBatch {
    const int32_t *pages, *kv_len, *cu_q;
    int64_t n_tokens;
    int n_seq, max_pages, max_q, max_kv;
};

// A batch whose sequences' leading tokens other rows read for them: the sequences with rows
// lead_cu[g] .. lead_cu[g + 1] leave out their first lead_len[g].  And that batch of
// leading tokens, every row of which sees all of its sequence's.
struct KvOwn : KvBatch {
    const int32_t *lead_cu, *lead_len;
    int n_lead;
};
struct KvLead : KvBatch {};

// A sequence's extent as the kernels use it: first row, new tokens, tokens.
struct KvSeq {
    int64_t row;  // of its first new token
    int q, n;
    bool ok;      // false: the bounds contradict what the arrays say of it (then
                  // q is within max_q and n is 0)
    int from;     // first token that the pass reads
};

#ifdef __HIPCC__
__device__ inline KvSeq kv_seq(const KvBatch& b, int s, int shift) {
    KvSeq r;
    const int64_t c0 = b.cu_q[s], c1 = b.cu_q[s + 1];
    r.n = b.kv_len[s];
    const bool rows = c0 >= 0 && c1 >= c0 && c1 <= b.n_tokens;
    r.row = rows ? c0 : 0;
    r.q = rows ? static_cast<int>(c1 - c0) : 0;
    r.ok = rows && r.q <= b.max_q && r.n >= 0 && r.n <= b.max_kv &&
           r.n <= (static_cast<int64_t>(b.max_pages) << shift);
    if (r.q > b.max_q) r.q = b.max_q;
    if (!r.ok) r.n = 0;
    r.from = 0;
    return r;
}

// As above, with what the group of its rows leaves out.  Lanes may ask for different sequences.
__device__ inline KvSeq kv_seq(const KvOwn& b, int s, int shift) {
    KvSeq r = kv_seq(static_cast<const KvBatch&>(b), s, shift);
    if (r.q == 0) return r;
    int g = 0;
    for (int len = b.n_lead; len > 1;) {
        const int half = len >> 1;
        if (b.lead_cu[g + half] <= r.row) {
            g += half;
            len -= half;
        } else {
            len = half;
        }
    }
    if (r.row < b.lead_cu[g] || r.row >= b.lead_cu[g + 1]) return r;
    r.from = max(b.lead_len[g], 0);
    // the group's rows are whole sequences, whose new tokens stand behind the prefix
    if (r.from && (r.row + r.q > b.lead_cu[g + 1] || r.n - r.q < r.from)) r.ok = false;
    if (!r.ok) r.n = r.from = 0;
    return r;
}

// The last s in [0, n) with key(s) <= x, for ascending keys of which the first is; the wave's
// lanes ask for one x together and look at 64 keys at once.
template <class F>
__device__ inline int last_at_most(int n, int64_t x, F key) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, len = n;
    while (len > 1) {
        const uint32_t step = (len + 63) / 64, i = lane * step;
        const uint64_t le = __ballot(i < len && key(static_cast<int>(lo + i)) <= x) | 1;
        const uint32_t at = (63 - __builtin_clzll(le)) * step;
        lo += at;
        len = min(step, len - at);
    }
    return static_cast<int>(lo);
}

// Page of token j of sequence s, or -1 where the table names none.
__device__ inline int kv_page(const KvBatch& b, const KvCache& c, int s, int j) {
    const int p = b.pages[static_cast<int64_t>(s) * b.max_pages + (j >> c.shift)];
    return p >= 0 && p < c.num_pages ? p : -1;
}

__device__ inline uint8_t* kv_block(const KvCache& c, int page, int head) {
    return c.base + (static_cast<int64_t>(page) * c.H + head) * c.block;
}
#endif

struct KvRows {
    const void* p;
    int64_t tok, head;  // strides in elements
};

struct Rotary;

// bits, D, dtype as checked by the entry points.  r: what keys are turned by, or null.
hipError_t kv_write(const KvCache& c, const KvBatch& b, int bits, int D, const KvRows& k,
                    const KvRows& v, int dtype, const Rotary* r, hipStream_t s);
hipError_t kv_read(const KvCache& c, const KvBatch& b, int bits, int D, void* k, void* v, int dtype,
                   hipStream_t s);

// slots: of each of the batch's rows, in f.
hipError_t kv_copy(const KvCache& f, const KvCache& c, const KvBatch& b, int bits, int D,
                   const int64_t* slots, hipStream_t s);
hipError_t kv_copy_pages(const KvCache& c, const int32_t* src, const int32_t* dst, int64_t n,
                         hipStream_t s);

struct KvAttend {
    KvRows q;
    int heads, G;    // query heads; of them per key/value head
    int dtype;       // of q and out: JHQ_BF16 or JHQ_F16
    float scale;
    int causal, window;
    void* out;
    int q16, out8;   // query rows start on 16 bytes, out on 8
    float* lse;
    float* work;
};
int64_t kv_attend_work(const KvCache& c, const KvBatch& b, int D, int G, int window);
hipError_t kv_attend(const KvCache& c, const KvBatch& b, int bits, int D, const KvAttend& a,
                     hipStream_t s);
// once: the prefix is read once whatever that costs, else where it pays.
int64_t kv_shared_work(const KvCache& c, const KvBatch& lead, const KvBatch& b, int D, int G, bool once);
hipError_t kv_attend_shared(const KvCache& c, const KvBatch& lead, const KvBatch& b, int bits, int D,
                            const KvAttend& a, bool once, hipStream_t s);

}  // namespace jhq
