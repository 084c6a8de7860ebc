// tg_i8_stream.hpp -- the 8-bit product of a few rows of A (up to 64) with a
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

// v without its first n bytes (16 and more: all), zeros behind.
__device__ __forceinline__ u32x4 shift_out(u32x4 v, int n) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    const u64x2 x = __builtin_bit_cast(u64x2, v);
    const int bits = n % 8 * 8;
    uint64_t lo = x[0] >> bits, hi = x[1] >> bits;
    if (bits != 0) lo |= x[1] << (64 - bits);
    if (n >= 8) lo = hi, hi = 0;
    if (n >= 16) lo = 0;
    return __builtin_bit_cast(u32x4, u64x2{lo, hi});
}

// The 16 bytes of a row of K from k on, zeros past its end.  load() takes the
// row's last 16 where the row ends among them or before, without a branch, so
// that several loads are on their way together; get() shifts them into place.
struct StreamTail {
    u32x4 v;
    int past;  // bytes of v that lie before k
    __device__ __forceinline__ void load(const int8_t* row, int k, int K) {
        if (K >= 16) {
            const int at = k < K - 16 ? k : K - 16;
            v = *reinterpret_cast<const u32x4_any*>(row + at);
            past = k - at;
        } else {
            v = u32x4{0, 0, 0, 0};
            for (int i = 0; i < K; ++i) v[i / 4] |= uint32_t(uint8_t(row[i])) << (8 * (i % 4));
            past = k;
        }
    }
    __device__ __forceinline__ u32x4 get() const { return shift_out(v, past); }
};

// The 16 bytes from byte `at` (0 ... 3) of v on; `next` is the word behind v.
__device__ __forceinline__ u32x4 align_words(u32x4 v, uint32_t next, int at) {
    return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], at), __builtin_amdgcn_alignbyte(v[2], v[1], at),
                 __builtin_amdgcn_alignbyte(v[3], v[2], at), __builtin_amdgcn_alignbyte(next, v[3], at)};
}

// 128 bytes of each of 16 rows in a wave, as lanes load them: lane l the
// 16-byte chunks l % 4 and l % 4 + 4 of row l / 4, so that four neighbouring
// lanes read 64 bytes of a row side by side.  get() hands them to the lanes as
// the matrix instruction has them (row l % 16, chunk l / 16).
//
// WORDS false: rows start at any address, and are read as the aligned words
// they lie in (an unaligned 16-byte load takes about as long as two aligned
// ones): `at` is the row's first byte in its first word, and a chunk's last
// bytes come from the next lane's first word.
template <bool WORDS>
struct StreamUnit {
    u32x4 v[2];
    uint32_t end;  // the word behind chunk 7, in that chunk's lanes
    __device__ __forceinline__ void load(const int8_t* row, int at) {
        const int c = threadIdx.x % 4;
        const int8_t* base = row - (WORDS ? 0 : at);
        v[0] = *reinterpret_cast<const u32x4_word*>(base + c * 16);
        v[1] = *reinterpret_cast<const u32x4_word*>(base + 64 + c * 16);
        // It holds the chunk's last bytes unless the row is aligned, so each
        // word read holds a byte of the row.
        if (!WORDS && c == 3) end = *reinterpret_cast<const uint32_t*>(base + (at != 0 ? 128 : 124));
    }
    static __device__ __forceinline__ u32x4 turn(u32x4 x) {
        const int from = (threadIdx.x % 16 * 4 + threadIdx.x % 64 / 16) * 4;
        u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = uint32_t(__builtin_amdgcn_ds_bpermute(from, int(x[i])));
        return y;
    }
    __device__ __forceinline__ void get(int at, u32x4 (&out)[2]) const {
        if constexpr (WORDS) {
            out[0] = turn(v[0]);
            out[1] = turn(v[1]);
        } else {
            // The first word of the next lane of four.
            constexpr int kNext = 1 | 2 << 2 | 3 << 4 | 0 << 6;
            const uint32_t n0 = uint32_t(__builtin_amdgcn_mov_dpp(int(v[0][0]), kNext, 15, 15, true));
            const uint32_t n1 = uint32_t(__builtin_amdgcn_mov_dpp(int(v[1][0]), kNext, 15, 15, true));
            const bool edge = threadIdx.x % 4 == 3;
            const uint32_t next[2] = {edge ? n1 : n0, edge ? end : n1};
#pragma unroll
            for (int i = 0; i < 2; ++i)
                out[i] = turn(align_words(v[i], next[i], at));
        }
    }
};

// A workgroup takes 16 rows of B (columns of C) and up to 16 * R rows of A;
// its W waves take the sum's 128-byte units in turn and add their sums in LDS.
// Bound by reading B: a wave has 2 KiB of B on their way, and the waves of a CU
// together cover HBM's latency.  Rows need no alignment: they go through
// registers.  A's are read again by every workgroup, from L2.  WORDS: rows
// start at multiples of four bytes.
template <int R, int W, bool WORDS, typename T>
__global__ __launch_bounds__(W * 64) void tg_i8_stream(StreamArgs p, TileStore<T> out) {
    typedef MmaAcc<Mma::I8>::type Acc;
    typedef StreamUnit<WORDS> Unit;
    __shared__ Acc part[R][W][64];
    const int t = threadIdx.x, lane = t % 64, wave = t / 64;
    const int n0 = int(blockIdx.x) * 16;
    // The lane's rows as it loads; those past the matrices repeat the last one
    // (their sums are not stored).
    const int lr = lane / 4, lc = lane % 4;
    const int8_t *pa[R], *pb = p.b + int64_t(n0 + lr < p.n ? n0 + lr : p.n - 1) * p.ldb;
    int at_a[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        pa[r] = p.a + int64_t(r * 16 + lr < p.m ? r * 16 + lr : p.m - 1) * p.lda;
        at_a[r] = int(reinterpret_cast<uintptr_t>(pa[r]) & 3);
    }
    const int at_b = int(reinterpret_cast<uintptr_t>(pb) & 3);
    Acc acc[R] = {};
    const int units = p.k / 128;
    // What does not need the sum is loaded before it, so that its latency is
    // not added to the end: the bytes behind the whole units, and scales.
    const bool last = wave == units % W && p.k % 128 != 0;
    StreamTail ta[R][2], tb[2];
    if (last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = units * 128 + i * 64 + lc * 16;
            tb[i].load(pb, k, p.k);
#pragma unroll
            for (int r = 0; r < R; ++r) ta[r][i].load(pa[r], k, p.k);
        }
    }
    // Wave r < R stores rows r * 16 ...: a lane four columns of one.
    const int li = wave * 16 + lane % 16, lg = lane / 16;
    const bool stores = wave < R && li < p.m;
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
        Unit xa[R], xb;
        xb.load(pb + u * 128, at_b);
#pragma unroll
        for (int r = 0; r < R; ++r) xa[r].load(pa[r] + u * 128, at_a[r]);
        u32x4 fa[2], fb[2];
        xb.get(at_b, fb);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            xa[r].get(at_a[r], fa);
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[r] = mma<Mma::I8>(fb[i], fa[i], acc[r]);
        }
    }
    if (last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 fb = Unit::turn(tb[i].get());
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] = mma<Mma::I8>(fb, Unit::turn(ta[r][i].get()), acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) part[r][wave][lane] = acc[r];
    __syncthreads();
    if (!stores) return;
    Acc sum = part[wave][0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += part[wave][w][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = n0 + lg * 4 + e;
        if (n >= p.n) continue;
        float v = float(sum[e]) * sa * sb[e];
        if (out.bias != nullptr) v += bias[e];
        out.c[int64_t(li) * p.n + n] = static_cast<T>(v);
    }
}

}  // namespace tg
