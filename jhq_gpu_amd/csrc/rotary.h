// rotary.h — turns of pairs by a token's position: the angle's arithmetic and the launcher of
// jhq_k_rotary.  Internal to rotary.hip and kvcache.hip.
#pragma once
#include "../../include/jhq.h"

#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>

namespace jhq {

// Pair i of a head turns by pos * turns[i] 2^-64 of a full turn, modulo one.
struct Rotary {
    const uint64_t* turns;
    int rot;          // elements in pairs
    int interleaved;  // pairs (2i, 2i + 1), else (i, i + rot / 2)
    float amp, sign;  // what cosines and sines are multiplied by, and sines beside it
};

// What is wrong with parameters, "" if nothing; parameters that are right, as kernels take them.
std::string rotary_wrong(const jhq_rotary* r);
Rotary rotary_of(const jhq_rotary& r, bool inverse);

#ifdef __HIPCC__
// Cosine and sine of pos * turn 2^-64 of a turn.  The product modulo 2^64 is exact whatever the
// position, which no float product is (2^20 radians have 2^-4 of error in float32): of the position only
// the frequency's own rounding is left, |pos| 2^-65 turns.  The upper 32 bits (what is cut off is below
// 2^-32 turns, 2^-29.3 radians) are cut into a quarter and a rest of at most pi / 4, which float32 leaves
// within 3 2^-24 of itself and whose sine and cosine are their series up to x^9 and
// x^10 (the next terms are below 2^-27 of the result).
__device__ inline void turn_of(uint64_t turn, int64_t pos, float& c, float& s) {
    const uint32_t ph = static_cast<uint32_t>(static_cast<uint64_t>(pos) * turn >> 32);
    const uint32_t quarter = (ph + 0x20000000u) >> 30;
    const float x = static_cast<float>(static_cast<int32_t>(ph - (quarter << 30))) *
                    1.46291807926715968e-9f;  // 2 pi 2^-32
    const float z = x * x;
    float a = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    a = fmaf(z, a, 8.33333333e-3f);
    a = fmaf(z, a, -1.66666667e-1f);
    a = fmaf(z * x, a, x);
    float b = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    b = fmaf(z, b, -1.38888889e-3f);
    b = fmaf(z, b, 4.16666667e-2f);
    b = fmaf(z, b, -0.5f);
    b = fmaf(z, b, 1.0f);
    const bool odd = quarter & 1;
    const float cc = odd ? a : b, ss = odd ? b : a;
    c = __uint_as_float(__float_as_uint(cc) ^ ((quarter + 1) << 30 & 0x80000000u));
    s = __uint_as_float(__float_as_uint(ss) ^ (quarter << 30 & 0x80000000u));
}
#endif

}  // namespace jhq
