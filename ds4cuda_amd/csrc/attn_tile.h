// attn_tile.h — the 32-key tile of the matrix-core attention kernels over the
// FP8 cache (prefill.hip, window_attn.hip): its FP8 bytes in registers, the
// dequantized f16 LDS tile, the key order inside a tile and the transposing
// reads of V.
#pragma once

#include "ds4hip_common.h"

namespace ds4hip {

constexpr int kD = 512;
constexpr int kRot = 64;
constexpr int kNope = kD - kRot;
constexpr int kTile = 32;            // keys per tile
constexpr int kRowB = 2 * kD + 32;   // one f16 row + 32 B
constexpr int kStageB = kTile * kRowB;
constexpr float kLog2e = 1.4426950408889634f;

// Byte-offset swizzle of row r of an f16 tile: rows 8..15 of every 16 swap
// the 16-byte halves of their 32-byte column groups. Chosen by measurement:
// 1056-byte rows with this swap ran 2% faster than 1040-byte rows and than
// unswapped 1056-byte rows, though a bank-conflict pattern test shows its
// 16-lane K reads 2-way conflicted and the unswapped form conflict-free.
__device__ inline uint32_t row_swz(int r) {
    return 16u * ((r >> 3) & 1);
}

// Tile-local key of S^T row / P column `idx` (0..31).
__device__ inline int pi_key(int idx) {
    const int h = idx >> 4, g = (idx >> 2) & 3, k = idx & 3;
    return 16 * h + 8 * (g >> 1) + (g & 1) + 2 * k;
}

__device__ inline uint32_t lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)p;
}

__device__ inline void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ inline float xmax_16_32(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float xsum_16_32(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Raw FP8 bytes of one tile held by one thread: row tid/8 of the tile, code
// bytes [56j, 56j+56) (j = tid%8, seven 8-byte groups, each inside one
// 64-dim block), the row's 8 scale exponents and tail granule j (f16 dims
// 448+8j .. +8).
struct Raw {
    uint2_t c[7];
    uint2_t e;
    uint4_t t;
};

// The thread's share (j = tid % 8) of cache row `row`.
__device__ inline void load_raw_row(const uint8_t *codes, const int8_t *sexp, const uint16_t *tail, long long row,
                                    int j, Raw &R) {
    const uint8_t *cp = codes + row * kNope + 56 * j;
#pragma unroll
    for (int i = 0; i < 7; ++i) R.c[i] = *reinterpret_cast<const uint2_t *>(cp + 8 * i);
    R.e = *reinterpret_cast<const uint2_t *>(sexp + row * 8);
    R.t = *reinterpret_cast<const uint4_t *>(tail + row * kRot + 8 * j);
}

template <bool kHi>
__device__ inline half2_t cvt2(uint32_t w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, scale, kHi);
}

// Dequantizes the thread's share of a tile into the f16 LDS tile.
__device__ inline void store_tile(uint8_t *stage, int tid, const Raw &R) {
    const int row = tid >> 3, j = tid & 7;
    uint8_t *rp = stage + row * kRowB;
    const uint32_t x = row_swz(row);
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        const int d = 56 * j + 8 * i;       // first dim of the group
        const int b = d >> 6;                       // its 64-dim block
        const uint32_t ew = b < 4 ? R.e[0] : R.e[1];
        const int e = (int)(int8_t)(ew >> (8 * (b & 3)));
        const float sc = __uint_as_float((uint32_t)(e + 127) << 23);
        const half2_t h0 = cvt2<false>(R.c[i][0], sc), h1 = cvt2<true>(R.c[i][0], sc);
        const half2_t h2 = cvt2<false>(R.c[i][1], sc), h3 = cvt2<true>(R.c[i][1], sc);
        *reinterpret_cast<half8_t *>(rp + ((2 * d) ^ x)) =
            half8_t{h0[0], h0[1], h1[0], h1[1], h2[0], h2[1], h3[0], h3[1]};
    }
    *reinterpret_cast<uint4_t *>(rp + ((2 * kNope + 16 * j) ^ x)) = R.t;
}

// V^T fragments of 4 of the wave's dim tiles (DT0 .. DT0+3): vb[i] holds,
// for lane (n, g), V[pi(4g+r)][128w+16(DT0+i)+n] then V[pi(16+4g+r)][...].
template <int DT0>
__device__ inline void read_vt4(uint32_t a0, uint32_t a1, half8_t *vb) {
    constexpr int o0 = 32 * DT0;
    uint2_t tb[8];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %9 offset:%10\n\t"
        "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %9 offset:%11\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %6, %8 offset:%13\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(tb[0]), "=&v"(tb[1]), "=&v"(tb[2]), "=&v"(tb[3]), "=&v"(tb[4]), "=&v"(tb[5]),
          "=&v"(tb[6]), "=&v"(tb[7])
        : "v"(a0), "v"(a1), "i"(o0), "i"(o0 + 32), "i"(o0 + 64), "i"(o0 + 96));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        vb[i] = __builtin_bit_cast(
            half8_t, uint4_t{tb[2 * i][0], tb[2 * i][1], tb[2 * i + 1][0], tb[2 * i + 1][1]});
}

}  // namespace ds4hip
