// tg_i8_stream.hpp -- the 8-bit product of a few rows of A (up to 16) with a
// weight matrix: every row of B is read once, straight into registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_tiles.hpp"

namespace tg {

struct StreamArgs {
    const int8_t* a;
    int64_t lda;
    const int8_t* b;
    int64_t ldb;
    int m, n, k;
};

// The 16 bytes of a row of K from k on; zeros past its end.  Where the row
// ends among them they are the row's last 16, shifted into place.
__device__ __forceinline__ u32x4 stream_tail(const int8_t* row, int k, int K) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    if (k >= K) return u32x4{0, 0, 0, 0};
    if (K >= 16) {
        const int past = k + 16 > K ? k + 16 - K : 0;  // 0 ... 15
        const u64x2 v = __builtin_bit_cast(u64x2, u32x4(*reinterpret_cast<const u32x4_any*>(row + k - past)));
        const int bits = past % 8 * 8;
        uint64_t lo = v[0] >> bits, hi = v[1] >> bits;
        if (bits != 0) lo |= v[1] << (64 - bits);
        if (past >= 8) lo = hi, hi = 0;
        return __builtin_bit_cast(u32x4, u64x2{lo, hi});
    }
    u32x4 v = {0, 0, 0, 0};
    for (int i = 0; i < K; ++i) v[i / 4] |= uint32_t(uint8_t(row[i])) << (8 * (i % 4));  // k is 0
    return v;
}

// 16 bytes of a row at any address, as the aligned words they lie in: an
// unaligned 16-byte load takes about as long as two aligned ones and four
// bytes more (M 1, N 5003, K 4099: 17 us so, 9 us as words).
template <bool WORDS>
struct StreamRaw {
    u32x4 v;
    __device__ __forceinline__ void load(const int8_t* p) { v = *reinterpret_cast<const u32x4_word*>(p); }
    __device__ __forceinline__ u32x4 get(int) const { return v; }
};
template <>
struct StreamRaw<false> {
    u32x4 v;
    uint32_t next;
    // The word behind the four holds the last bytes unless p is aligned, so
    // each word read holds a byte of the row.
    __device__ __forceinline__ void load(const int8_t* p) {
        const int at = int(reinterpret_cast<uintptr_t>(p) & 3);
        const int8_t* base = p - at;
        v = *reinterpret_cast<const u32x4_word*>(base);
        next = *reinterpret_cast<const uint32_t*>(base + (at != 0 ? 16 : 12));
    }
    __device__ __forceinline__ u32x4 get(int at) const {
        return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], at), __builtin_amdgcn_alignbyte(v[2], v[1], at),
                     __builtin_amdgcn_alignbyte(v[3], v[2], at), __builtin_amdgcn_alignbyte(next, v[3], at)};
    }
};

// A workgroup takes 16 rows of B (columns of C) and up to 16 rows of A; its W
// waves take the sum's 128-byte units in turn and add their sums in LDS.
// Bound by reading B: a wave has two loads of 1 KiB of B in flight, and the 32
// waves of a CU together cover HBM's latency (N = K = 8192, M = 1: 15.0 us,
// 4.5 TB/s, with 16 waves a workgroup, 16.7 with 8; four loads a wave or 32
// rows of B a workgroup are slower, 17 to 25 us at M = 13).  Fragments come
// straight from memory (a lane's 16 bytes at any address), so rows need no
// alignment; A's are read again by every workgroup, from L2.  WORDS: rows
// start at multiples of four bytes.
template <int W, bool WORDS, typename T>
__global__ __launch_bounds__(W * 64) void tg_i8_stream(StreamArgs p, TileStore<T> out) {
    typedef MmaAcc<Mma::I8>::type Acc;
    __shared__ Acc part[W][64];
    const int t = threadIdx.x, lane = t % 64, wave = t / 64, li = lane % 16, lg = lane / 16;
    const int n0 = int(blockIdx.x) * 16;
    // Rows past the matrices repeat their last one; their sums are not stored.
    const int8_t* pa = p.a + int64_t(li < p.m ? li : p.m - 1) * p.lda;
    const int8_t* pb = p.b + int64_t(n0 + li < p.n ? n0 + li : p.n - 1) * p.ldb;
    const int at_a = int(reinterpret_cast<uintptr_t>(pa) & 3), at_b = int(reinterpret_cast<uintptr_t>(pb) & 3);
    Acc acc = {};
    const int units = p.k / 128;
    // What does not need the sum is loaded before it, so that its latency is
    // not added to the end: the bytes behind the whole units, and scales.
    const bool last = wave == units % W;
    u32x4 ta[2], tb[2];
    if (last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            tb[i] = stream_tail(pb, units * 128 + i * 64 + lg * 16, p.k);
            ta[i] = stream_tail(pa, units * 128 + i * 64 + lg * 16, p.k);
        }
    }
    const bool stores = wave == 0 && li < p.m;
    float sa = 0, sb[4] = {}, bias[4] = {};
    if (stores) {
        sa = out.a_scale[li];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + lg * 4 + e < p.n ? n0 + lg * 4 + e : p.n - 1;
            sb[e] = out.b_scale[n];
            if (out.bias != nullptr) bias[e] = to_f32(out.bias[n]);
        }
    }
    for (int u = wave; u < units; u += W) {
        StreamRaw<WORDS> xa[2], xb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            xb[i].load(pb + u * 128 + i * 64 + lg * 16);
            xa[i].load(pa + u * 128 + i * 64 + lg * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) acc = mma<Mma::I8>(xb[i].get(at_b), xa[i].get(at_a), acc);
    }
    if (last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) acc = mma<Mma::I8>(tb[i], ta[i], acc);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (!stores) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc += part[w][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = n0 + lg * 4 + e;
        if (n >= p.n) continue;
        float v = float(acc[e]) * sa * sb[e];
        if (out.bias != nullptr) v += bias[e];
        out.c[int64_t(li) * p.n + n] = static_cast<T>(v);
    }
}

}  // namespace tg
