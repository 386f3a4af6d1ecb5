// Attention over packed token sequences: the parts its kernels share.
//
// Row packing.  The G = Hq / Hk query heads that share a key/value head are rows of ONE problem: row r of a sequence is token r / G, head
// r % G, so a tile of rows reads each key tile once for all heads of the group and a causal tile spans 1/G of the tokens.
//
// Orientation.  A wave owns 32 columns (query rows in the forward and dQ kernels, keys in the dK/dV kernel), one per lane pair
// (lane, lane + 32), and every product is built with that column on the matrix instruction's N axis:
//   S^T = A * B      A: a 32-row tile of the OTHER side from LDS, B: the wave's own columns, held in registers
//   acc^T += X^T * P    P: the C registers of the product above, used as the next B operand as they are -- C register i of lane half h is
//                       row 8 (i / 4) + 4 h + i % 4, and the contraction runs over the rows in whatever order both operands name them, so
//                       X is read in that order (bf16: transposing LDS reads; fp32: one row and 32 columns per read)
// No exchange between lanes is needed but one maximum across the two lane halves per tile.
//
// LDS tiles are [rows][DP] in 16-byte chunks, chunk c of a row at place c ^ swizzle(row): 16 consecutive rows at one chunk (operand A) and
// 4 rows x 64 bytes (transposed operand X) then touch all 64 banks once.
#pragma once
#include "common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct AttnGeom {
    const int* off_q;       // [B + 1]
    const int* off_k;       // [B + 1]
    const int* k_len;       // [B] used rows of each key sequence, or null
    int B, Nq, Nk, Hq, Hk, G, D;
    int causal, fill;
    float c;                // log2(e) / temperature
    float scale;            // 1 / temperature
};
struct AttnTensor { const void* p; long long ts, hs; };

struct AttnSeq { int q0, lq, k0, lk, room; };

// Sequence b.  Offsets come from device memory, so they are clamped into the tensors here: a wrong offset gives wrong rows, never an access
// outside
__device__ __forceinline__ AttnSeq attn_seq(const AttnGeom& g, int b) {
    AttnSeq s;
    s.q0 = min(max(g.off_q[b], 0), g.Nq);
    s.lq = min(max(g.off_q[b + 1], s.q0), g.Nq) - s.q0;
    s.k0 = min(max(g.off_k[b], 0), g.Nk);
    s.room = min(max(g.off_k[b + 1], s.k0), g.Nk) - s.k0;
    s.lk = g.k_len ? min(max(g.k_len[b], 0), s.room) : s.room;
    return s;
}

// Tiles of `1 << shift` rows over sequences of per * (off[b + 1] - off[b]) rows.  Sequence b owns the slots from
// floor(per * off[b] / rows) + b on: floor(x + y) + 1 >= floor(x) + ceil(y), so each sequence has as many as it needs, the total is known
// without reading the offsets, and no pass over them is needed.  64 lanes probe at a time.
__device__ __forceinline__ int attn_slot(const int* off, int b, int N, int per, int shift) {
    return (int)(((long long)min(max(off[b], 0), N) * per) >> shift) + b;
}
__device__ __forceinline__ bool attn_find(const int* off, int B, int N, int per, int shift, int slot, int& b, int& tile) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = B;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool in = lane * step < n && attn_slot(off, lo + lane * step, N, per, shift) <= slot;
        const int cnt = max(__popcll(__ballot(in)), 1);
        lo += (cnt - 1) * step;
        n = min(step, n - (cnt - 1) * step);
    }
    b = lo;
    tile = slot - attn_slot(off, lo, N, per, shift);
    return tile >= 0;
}
static inline int attn_slots(long long rows, int B, int shift) { return (int)(rows >> shift) + B; }

template <typename T> struct AttnElem;
template <> struct AttnElem<float> { typedef f32x4 Frag; static constexpr int EPC = 4; };
template <> struct AttnElem<__bf16> { typedef bf16x8 Frag; static constexpr int EPC = 8; };

template <typename T, int DP> struct AttnTile {
    typedef typename AttnElem<T>::Frag Frag;
    static constexpr int EPC = AttnElem<T>::EPC;          // elements per 16-byte chunk
    static constexpr int NCH = DP / EPC;                  // chunks per row
    static constexpr int RB = NCH * 16;                   // bytes per row
    static constexpr int KS = NCH / 2;                    // operand steps over DP: a step is one chunk of each lane half
    static constexpr int DB = DP / 32;                    // 32-wide blocks of DP

    static __device__ __forceinline__ int swizzle(int row) {
        if (NCH >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        if (NCH == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        return (row >> 2) & 3;
    }
    static __device__ __forceinline__ int place(int row, int chunk) { return row * RB + ((chunk ^ swizzle(row)) << 4); }

    // operand A (or B) of step s for row `row` of a tile
    static __device__ __forceinline__ Frag frag(const char* tile, int row, int s, int h) {
        return *reinterpret_cast<const Frag*>(tile + place(row, 2 * s + h));
    }

    // 16 bytes of a row in global memory, zeros behind D.  VEC: rows start at 16-byte boundaries and D fills whole chunks
    template <bool VEC> static __device__ __forceinline__ Frag fetch(const T* row, int chunk, int D) {
        Frag f = {};
        if (VEC) {
            if (chunk * EPC < D) f = *reinterpret_cast<const Frag*>(row + chunk * EPC);
        } else {
#pragma unroll
            for (int i = 0; i < EPC; ++i)
                if (chunk * EPC + i < D) f[i] = row[chunk * EPC + i];
        }
        return f;
    }
};

// acc (32 x 32) += A * B over one step
__device__ __forceinline__ void attn_mma(f32x16& acc, const bf16x8& a, const bf16x8& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void attn_mma(f32x16& acc, const f32x4& a, const f32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
}

// The C registers of a 32-row product as the B operand of the next one (bf16: rounded once, to nearest even)
template <typename T> struct AttnProb;
template <> struct AttnProb<__bf16> {
    bf16x8 v[2];
    __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x8 t;
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = p[8 * u + i];
            v[u] = __builtin_convertvector(t, bf16x8);
        }
    }
};
template <> struct AttnProb<float> {
    f32x16 v;
    __device__ __forceinline__ void set(const f32x16& p) { v = p; }
};

// acc[32 of DP][32 columns] += X^T * P over the 32 rows row0 .. row0 + 31 of the tile X
template <int DP> __device__ __forceinline__ void attn_mma_t(f32x16& acc, const char* tile, int row0, int db, int lane, const AttnProb<__bf16>& p) {
    typedef AttnTile<__bf16, DP> L;
    const int g = lane >> 4, l = lane & 15;
    const int chunk = db * 4 + (g & 1) * 2 + ((l & 3) >> 1), low = (l & 1) * 8;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int row = row0 + 16 * u + 4 * (g >> 1) + (l >> 2);
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + L::place(row, chunk) + low));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + L::place(row + 8, chunk) + low));
        const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
        const bf16x8 f = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, p.v[u], acc, 0, 0, 0);
    }
}
template <int DP> __device__ __forceinline__ void attn_mma_t(f32x16& acc, const char* tile, int row0, int db, int lane, const AttnProb<float>& p) {
    typedef AttnTile<float, DP> L;
    const int col = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = row0 + 8 * (i / 4) + 4 * h + i % 4;
        const float x = *reinterpret_cast<const float*>(tile + L::place(row, db * 8 + (col >> 2)) + (col & 3) * 4);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p.v[i], acc, 0, 0, 0);
    }
}

// A block's share of a tile on its way from global memory to LDS: fetched into registers while the previous tile is computed on
template <typename T, int DP, int ROWS, int NT, bool VEC> struct AttnStage {
    typedef AttnTile<T, DP> L;
    static constexpr int CNT = (ROWS * L::NCH + NT - 1) / NT;
    typename L::Frag f[CNT];
    // rows row0 ..: those behind `last` repeat it (their products are masked)
    __device__ __forceinline__ void fetch(const T* base, long long ts, int row0, int last, int D) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int c = threadIdx.x + i * NT;
            if ((ROWS * L::NCH) % NT && c >= ROWS * L::NCH) break;
            f[i] = L::template fetch<VEC>(base + (size_t)min(row0 + c / L::NCH, last) * ts, c % L::NCH, D);
        }
    }
    // packed rows: token r / G, head r % G
    __device__ __forceinline__ void fetch_packed(const T* base, long long ts, long long hs, int row0, int last, int G, int D) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int c = threadIdx.x + i * NT;
            if ((ROWS * L::NCH) % NT && c >= ROWS * L::NCH) break;
            const unsigned r = min(row0 + c / L::NCH, last), t = r / (unsigned)G;
            f[i] = L::template fetch<VEC>(base + (size_t)t * ts + (size_t)(r - t * G) * hs, c % L::NCH, D);
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int c = threadIdx.x + i * NT;
            if ((ROWS * L::NCH) % NT && c >= ROWS * L::NCH) break;
            *reinterpret_cast<typename L::Frag*>(tile + L::place(c / L::NCH, c % L::NCH)) = f[i];
        }
    }
};

// column `col`'s accumulators acc[DB] (d = 32 db + 8 (i / 4) + 4 h + i % 4) times f into a row of D elements
template <typename T, int DB> __device__ __forceinline__ void attn_store_row(T* row, const f32x16 (&acc)[DB], float f, int h, int D) {
    typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = db * 32 + q * 8 + h * 4;
            T4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (T)(acc[db][4 * q + i] * f);
            if ((D & 3) == 0) {
                if (d < D) __builtin_memcpy(__builtin_assume_aligned(row + d, sizeof(T) * 4), &v, sizeof(v));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < D) row[d + i] = v[i];
            }
        }
}

__device__ __forceinline__ float attn_other_half(float x) { return __shfl_xor(x, 32); }

// Rows of the tensor that belong to no sequence, [0, first) and [behind, N), shared out over the grid: `width` zeros each (and -inf in `lse`)
template <typename T> __device__ __forceinline__ void attn_fill_outside(const int* off, int B, int N, T* out, long long ts, long long hs, int H,
                                                                        int D, float* lse, int block, int blocks) {
    const int first = min(max(off[0], 0), N), behind = min(max(off[B], first), N);
    const int rows = first + N - behind;
    for (int i = block; i < rows; i += blocks) {
        const int r = i < first ? i : behind + i - first;
        for (int e = threadIdx.x; e < H * D; e += blockDim.x) out[(size_t)r * ts + (size_t)(e / D) * hs + e % D] = (T)0.f;
        if (lse)
            for (int e = threadIdx.x; e < H; e += blockDim.x) lse[(size_t)r * H + e] = -INFINITY;
    }
}

// host side (packed_attn.hip)
int attn_geom(AttnGeom& g, const int* off_q, const int* off_k, const int* k_len, float temperature, int causal, int B, int Nq, int Nk, int Hq,
              int Hk, int D, int act);
bool attn_aligned(const AttnTensor* t, int n, int D, int act);
