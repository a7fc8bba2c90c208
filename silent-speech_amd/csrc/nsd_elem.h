// Element types of the AR head's kernels (fp32 or bf16 storage, arithmetic in fp32), their 16-byte pieces, and wave-wide
// reductions (gfx950, wave64).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "nsd_device.h"

namespace {

struct BF16 { uint16_t b; };

template <class T> NSD_D float to_f(T v);
template <> NSD_D float to_f<float>(float v) { return v; }
template <> NSD_D float to_f<BF16>(BF16 v) { return __uint_as_float((uint32_t)v.b << 16); }

template <class T> NSD_D T from_f(float v);
template <> NSD_D float from_f<float>(float v) { return v; }
template <> NSD_D BF16 from_f<BF16>(float v)
{
    uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return BF16{(uint16_t)((u >> 16) | 0x40u)};     // NaN stays NaN
    u += 0x7fffu + ((u >> 16) & 1u);                                                   // round to nearest even
    return BF16{(uint16_t)(u >> 16)};
}

// sixteen bytes of a row as floats: 4 (fp32) or 8 (bf16) elements
template <class T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int N = 4;
    NSD_D static void unpack(const uint4 &v, float (&o)[8])
    {
        o[0] = __uint_as_float(v.x); o[1] = __uint_as_float(v.y); o[2] = __uint_as_float(v.z); o[3] = __uint_as_float(v.w);
    }
    NSD_D static void load(const float *p, float (&o)[8]) { unpack(*reinterpret_cast<const uint4 *>(p), o); }
};
template <> struct Vec16<BF16> {
    static constexpr int N = 8;
    NSD_D static void unpack(const uint4 &v, float (&o)[8])
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = __uint_as_float(w[i] << 16);
            o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    NSD_D static void load(const BF16 *p, float (&o)[8]) { unpack(*reinterpret_cast<const uint4 *>(p), o); }
};

// Wave-wide maximum / sum, the same value in every lane.  Inside a row of 16 lanes the butterfly runs on DPP register
// moves (after the distance-1 and -2 steps a quad is uniform, so the mirrored lane of the other quad / half carries
// what the lane at distance 4 / 8 carries); the four row results meet through scalar registers.  No LDS-crossbar
// permutes: they cost an address, an LDS instruction and its latency per step.
NSD_D float nsd_dpp_row_mirror(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));
}
NSD_D float row_lane(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
NSD_D float wave_max_f(float v)
{
    v = fmaxf(v, nsd_dpp_xor1(v));
    v = fmaxf(v, nsd_dpp_xor2(v));
    v = fmaxf(v, nsd_dpp_half_mirror(v));
    v = fmaxf(v, nsd_dpp_row_mirror(v));
    return fmaxf(fmaxf(row_lane(v, 0), row_lane(v, 16)), fmaxf(row_lane(v, 32), row_lane(v, 48)));
}
NSD_D float wave_sum_f(float v)
{
    v = v + nsd_dpp_xor1(v);
    v = v + nsd_dpp_xor2(v);
    v = v + nsd_dpp_half_mirror(v);
    v = v + nsd_dpp_row_mirror(v);
    return (row_lane(v, 0) + row_lane(v, 16)) + (row_lane(v, 32) + row_lane(v, 48));
}

// sixteen bytes of a row written from floats, rounded to the element type
template <class T> struct Store16;
template <> struct Store16<float> {
    NSD_D static void store(float *p, const float (&v)[8]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct Store16<BF16> {
    NSD_D static void store(BF16 *p, const float (&v)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)from_f<BF16>(v[2 * i]).b | ((uint32_t)from_f<BF16>(v[2 * i + 1]).b << 16);
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

} // namespace
