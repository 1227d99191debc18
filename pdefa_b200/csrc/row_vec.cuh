// 16-byte vectors of rows that start anywhere in memory: aligned accesses and a shift by the
// row's offset within 16 bytes, instead of accesses of one element each.
#pragma once

#include "device_common.cuh"

namespace pb {

// Bytes 4 * words + bits / 8 and the 15 after it of the 32 bytes lo, hi.
__device__ __forceinline__ uint4 shift_pair(const uint4& lo, const uint4& hi, int words, int bits) {
    uint32_t s[5];
    switch (words) {
        case 0: s[0] = lo.x; s[1] = lo.y; s[2] = lo.z; s[3] = lo.w; s[4] = hi.x; break;
        case 1: s[0] = lo.y; s[1] = lo.z; s[2] = lo.w; s[3] = hi.x; s[4] = hi.y; break;
        case 2: s[0] = lo.z; s[1] = lo.w; s[2] = hi.x; s[3] = hi.y; s[4] = hi.z; break;
        default: s[0] = lo.w; s[1] = hi.x; s[2] = hi.y; s[3] = hi.z; s[4] = hi.w; break;
    }
    return make_uint4(__funnelshift_r(s[0], s[1], bits), __funnelshift_r(s[1], s[2], bits),
                      __funnelshift_r(s[2], s[3], bits), __funnelshift_r(s[3], s[4], bits));
}

// Vector v of a row of n elements of T: elements v * 16 / sizeof(T) and on, `fill` (the bits of
// one element) past the end. Nothing outside the row is read.
template <typename T>
struct RowLoader {
    static constexpr uint32_t kPer = 16 / sizeof(T);
    const T* row;
    uint32_t n;
    const uint4* base;          // the aligned vector that holds the row's first element
    int words, bits;            // the row's offset in it
    uint32_t fill;
    __device__ __forceinline__ RowLoader(const T* r, uint32_t len, uint32_t f) : row(r), n(len), fill(f) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(r) & 15);
        base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(r) - off);
        words = (int)(off >> 2);
        bits = (int)(off & 3) * 8;
    }
    __device__ __forceinline__ bool aligned() const { return (words | bits) == 0; }
    __device__ __forceinline__ uint32_t whole() const { return n / kPer; }      // vectors without elements past the end
    // vectors 1 .. inner() - 1 have both their aligned ones inside the row
    __device__ __forceinline__ uint32_t inner() const { return n / kPer > 0 ? n / kPer - 1 : 0; }
    __device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi) const { return shift_pair(lo, hi, words, bits); }
    __device__ __forceinline__ uint4 operator()(uint32_t v) const {
        const uint32_t i = v * kPer;
        if (aligned() && i + kPer <= n) return base[v];
        // both vectors lie inside the row unless v is its first or its last
        if (v > 0 && i + 2 * kPer <= n) return shift_pair(base[v], base[v + 1], words, bits);
        uint32_t w[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (sizeof(T) == 4) {
                w[j] = i + j < n ? reinterpret_cast<const uint32_t*>(row)[i + j] : fill;
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
                w[j] = (i + 2 * j < n ? h[i + 2 * j] : fill) | ((i + 2 * j + 1 < n ? h[i + 2 * j + 1] : fill) << 16);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

}  // namespace pb
