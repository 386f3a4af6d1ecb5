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
#include <limits.h>

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
    int causal, fill, sorted;
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
    return tile >= 0 && tile <= (int)(((long long)N * per) >> shift);      // more only if the offsets decrease: no row number may wrap
}
// The same tiles in descending order of their causal work, for a few long sequences: with tiles in the order of the sequences a long one
// that comes late keeps some blocks busy long after the others have ended (five sequences of 2832 to 5000 tokens, 16/4 heads of 128, dK/dV:
// 1210 -> 950 us).  Tile j, counted from its sequence's heaviest, has v = lk * G - rows * j (rows of the group it meets, up
// to a constant); the block numbered n looks for the largest v that at least n + 1 tiles reach -- 64 candidates at a time, one per lane --
// and among the tiles that have it takes them in the order of the sequences.
constexpr int ATTN_SORT_MAX_B = 64;
template <bool KEYS> __device__ __forceinline__ bool attn_find_sorted(const AttnGeom& g, int rows, int n, int& b, int& tile) {
    __shared__ int top[ATTN_SORT_MAX_B], tiles[ATTN_SORT_MAX_B];
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < (unsigned)g.B) {
        const AttnSeq s = attn_seq(g, threadIdx.x);
        top[threadIdx.x] = s.lk * g.G;
        tiles[threadIdx.x] = ((KEYS ? s.room : s.lq * g.G) + rows - 1) / rows;
    }
    __syncthreads();
    const int unit = KEYS ? rows * g.G : rows;
    int lo = INT_MAX, hi = INT_MIN, total = 0;
    for (int i = 0; i < g.B; ++i) {
        if (!tiles[i]) continue;
        total += tiles[i];
        hi = max(hi, top[i]);
        lo = min(lo, top[i] - unit * (tiles[i] - 1));
    }
    if (n >= total) return false;
    // tiles with v >= x
    auto reach = [&](int x) {
        int c = 0;
        for (int i = 0; i < g.B; ++i)
            if (top[i] >= x) c += min(tiles[i], (top[i] - x) / unit + 1);
        return c;
    };
    // reach(lo) = total > n: the largest x in [lo, hi] with reach(x) > n
    while (lo < hi) {
        const int step = (int)(((unsigned)hi - (unsigned)lo) / 64u) + 1;
        const long long x = (long long)lo + (long long)step * lane;
        const int cnt = __popcll(__ballot(x <= hi && reach((int)x) > n));      // lane 0 always
        lo += step * (cnt - 1);
        hi = (int)min((long long)hi, (long long)lo + step - 1);
    }
    n -= reach(lo + 1);
    for (b = 0; b < g.B; ++b) {
        const int d = top[b] - lo;
        if (d >= 0 && d % unit == 0 && d / unit < tiles[b] && n-- == 0) break;
    }
    if (b >= g.B) return false;
    tile = KEYS ? (top[b] - lo) / unit : tiles[b] - 1 - (top[b] - lo) / unit;
    return true;
}
// Fewer than four blocks of `rows` rows per CU: CUs with one block more than others set the time.  Blocks of half as many rows then, whose
// waves pair up and share the keys of each tile (two sequences of 4096 and 1587 tokens, 8 heads of 32, fp32: forward
// 254 -> 225 us, dQ 358 -> 313 us)
static inline bool attn_few_blocks(const AttnGeom& g, int rows) { return (((long long)g.Nq * g.G / rows) + g.B) * g.Hk < 1024; }
// Sequences of up to 64 rows on average: blocks of two waves and tiles of 32 keys, four or more per CU, where larger blocks would have most of
// their waves without rows (1500 causal series of up to 64 tokens, 4 heads of 128, bf16: forward 187 -> 67 us, dQ 243 -> 97; up to 60, 8/4
// heads of 64: 66 -> 44 and 90 -> 70; fp32, 4 heads of 128: 393 -> 214 and 487 -> 263).  Up to 48 keys: blocks of 64 keys in dK/dV (those of 64,
// bf16: 184 -> 104 us, fp32: 450 -> 263; 4 heads of 128, bf16, whose tiles of rows are half as long then: 209 -> 121).  Where a launch has few
// blocks, the half-size blocks above share the keys instead.
static inline bool attn_low_rows(const AttnGeom& g) { return (long long)g.Nq * g.G <= 64ll * g.B; }
static inline bool attn_low_keys(const AttnGeom& g) { return g.Nk <= 48ll * g.B; }
// Sorting costs a block about 2 us: for causal sequences of at least four tiles on average
static inline bool attn_sorts(const AttnGeom& g, long long rows, int per_tile) {
    return g.causal && g.B <= ATTN_SORT_MAX_B && rows / per_tile >= 4ll * g.B && (long long)g.Nk * g.G < (1ll << 29) && (long long)g.G * per_tile < (1 << 20);
}
static inline int attn_slots(long long rows, int B, int shift) { return (int)(rows >> shift) + B; }
// a launch's threads are counted in 32 bits
static inline bool attn_grid(long long blocks, int threads) { return blocks * threads <= 0xffffffffll; }

// fp32 on the bf16 matrix units: x = x0 + x1 + x2 exactly to 24 bits, each rounded to bf16 from what the ones before leave, and
//   a b = a0 b0 + a0 b1 + a1 b0 + a1 b1 + a0 b2 + a2 b0      (left out: a1 b2 + a2 b1 of at most 2 * 2^-24 |a b|, two half steps of fp32)
// -- six products at 16 times the rate of v_mfma_f32_32x32x2_f32.  A launch before lays the inputs out as rows [3][D rounded up to 8]
// (attn_planes below); P and dS are taken apart in registers.
struct AttnThree {};

template <typename T> struct AttnElem;
template <> struct AttnElem<float> { typedef f32x4 Frag; typedef float In, Out; static constexpr int EPC = 4; static constexpr bool THREE = false; };
template <> struct AttnElem<__bf16> { typedef bf16x8 Frag; typedef __bf16 In, Out; static constexpr int EPC = 8; static constexpr bool THREE = false; };
template <> struct AttnElem<AttnThree> { typedef bf16x8 Frag; typedef __bf16 In; typedef float Out; static constexpr int EPC = 8; static constexpr bool THREE = true; };

template <typename T, int DP> struct AttnTile {
    typedef typename AttnElem<T>::Frag Frag;
    typedef typename AttnElem<T>::In In;
    static constexpr bool THREE = AttnElem<T>::THREE;
    static constexpr int EPC = AttnElem<T>::EPC;          // elements per 16-byte chunk
    static constexpr int NCH = DP / EPC;                  // chunks per row (and part)
    static constexpr int CPR = THREE ? 3 * NCH : NCH;     // chunks of a row in LDS
    static constexpr int RB = CPR * 16;                   // bytes per row
    static constexpr int KS = NCH / 2;                    // operand steps over DP: a step is one chunk of each lane half
    // waves per SIMD the kernels are compiled for: no more registers than 512 / WAVES, so that the accumulators stay where vector
    // instructions reach them (the compiler moves them to and fro otherwise)
    static constexpr int WAVES = THREE ? (DP <= 32 ? 3 : 2) : RB <= 128 ? 3 : RB <= 256 ? 2 : 1;
    static constexpr int DB = DP < 32 ? 1 : DP / 32;      // 32-wide blocks of DP (DP = 16: half a block, its other half repeats the first)

    static __device__ __forceinline__ int swizzle(int row) {
        if (NCH >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        if (NCH == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        if (NCH == 4) return (row >> 2) & 3;
        return (row >> 3) & 1;
    }
    static __device__ __forceinline__ int place(int row, int chunk, int part = 0) { return row * RB + part * NCH * 16 + ((chunk ^ swizzle(row)) << 4); }

    // operand A (or B) of step s for row `row` of a tile
    static __device__ __forceinline__ Frag frag(const char* tile, int row, int s, int h, int part = 0) {
        return *reinterpret_cast<const Frag*>(tile + place(row, 2 * s + h, part));
    }

    // 16 bytes of a row in global memory, zeros behind D.  VEC: rows start at 16-byte boundaries and D fills whole chunks
    template <bool VEC> static __device__ __forceinline__ Frag fetch(const In* row, int chunk, int D, int part = 0) {
        Frag f = {};
        if (THREE) {
            if (chunk * EPC < D) f = *reinterpret_cast<const Frag*>(row + part * ((D + 7) & ~7) + chunk * EPC);
        } else if (VEC) {
            if (chunk * EPC < D) f = *reinterpret_cast<const Frag*>(row + chunk * EPC);
        } else {
#pragma unroll
            for (int i = 0; i < EPC; ++i)
                if (chunk * EPC + i < D) f[i] = row[chunk * EPC + i];
        }
        return f;
    }
    // what belongs at place c of a tile: chunk and part of row c / CPR
    static __device__ __forceinline__ int chunk_at(int c) { return (c % CPR % NCH) ^ swizzle(c / CPR); }
    static __device__ __forceinline__ int part_at(int c) { return c % CPR / NCH; }
};

// The two buffers of key and value tiles of a block, in ONE object: once nobody needs the tiles any more, the waves that shared the keys add
// their sums through all of it (bf16 heads of 128: 64 KB, which the keys' buffers alone would not hold)
template <typename T, int DP, int TK> struct AttnBuffers {
    typedef AttnTile<T, DP> L;
    char k[2][TK * L::RB], v[2][TK * L::RB];
    // accumulators of group `i` of GROUPS pairs of waves: [DB * 16][64 lanes]
    template <int GROUPS> __device__ __forceinline__ float* join(int i) {
        static_assert(sizeof(float) * GROUPS * L::DB * 16 * 64 <= sizeof(AttnBuffers), "the tiles do not hold the sums of the waves that join");
        return (float*)this + i * (L::DB * 16 * 64);
    }
};

// Operands are fetched from LDS in one go and used after it (`attn_fence` keeps the compiler from sinking each read to its use, where
// every product waits for the latency of its own operand)
__device__ __forceinline__ void attn_fence() { __builtin_amdgcn_sched_barrier(0); }

// operand A of a 32-row product: all of a row's chunks this lane half holds
template <typename T, int DP> struct AttnRows {
    typedef AttnTile<T, DP> L;
    static constexpr int PARTS = L::THREE ? 3 : 1;
    typename L::Frag f[PARTS][L::KS];
    __device__ __forceinline__ void fetch(const char* tile, int row, int h) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int i = 0; i < L::KS; ++i) f[p][i] = L::frag(tile, row, i, h, p);
    }
    // 16 bytes at a time from a row in global memory
    template <bool VEC> __device__ __forceinline__ void fetch_global(const typename L::In* row, int h, int D) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int i = 0; i < L::KS; ++i) f[p][i] = L::template fetch<VEC>(row, 2 * i + h, D, p);
    }
    // sum of this half's products with another row
    __device__ __forceinline__ float dot(const AttnRows& o) const {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < L::KS; ++i)
#pragma unroll
            for (int e = 0; e < L::EPC; ++e) d = fmaf((float)f[0][i][e], (float)o.f[0][i][e], d);
        return d;
    }
};

__device__ __forceinline__ void attn_mma(f32x16& acc, const bf16x8& a, const bf16x8& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void attn_mma(f32x16& acc, const f32x4& a, const f32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
}
// the six products of two numbers in three parts, small ones first
__device__ __forceinline__ void attn_mma_three(f32x16& acc, const bf16x8& a0, const bf16x8& a1, const bf16x8& a2, const bf16x8& b0, const bf16x8& b1,
                                               const bf16x8& b2) {
    attn_mma(acc, a2, b0);
    attn_mma(acc, a0, b2);
    attn_mma(acc, a1, b1);
    attn_mma(acc, a1, b0);
    attn_mma(acc, a0, b1);
    attn_mma(acc, a0, b0);
}
// acc (32 rows of A x 32 columns of B) = A * B
template <typename T, int DP> __device__ __forceinline__ f32x16 attn_product(const AttnRows<T, DP>& a, const AttnRows<T, DP>& b) {
    f32x16 acc = (f32x16)(0.f);
#pragma unroll
    for (int i = 0; i < AttnTile<T, DP>::KS; ++i) {
        if constexpr (AttnTile<T, DP>::THREE) attn_mma_three(acc, a.f[0][i], a.f[1][i], a.f[2][i], b.f[0][i], b.f[1][i], b.f[2][i]);
        else attn_mma(acc, a.f[0][i], b.f[0][i]);
    }
    return acc;
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
template <> struct AttnProb<AttnThree> {
    bf16x8 v[3][2];
    __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x8 t;
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = p[8 * u + i];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                v[k][u] = __builtin_convertvector(t, bf16x8);
                if (k < 2) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) t[i] -= (float)v[k][u][i];
                }
            }
        }
    }
};

// The C registers of a 32-row product on their way through LDS from one wave to another, lane by lane, conflict-free.  With bf16 storage the
// upper three bytes of each cross, 16 significant bits: all four do not fit beside the tiles, and as bf16 P would take the rounding that
// dS gets anyway a second time (dK's error against 64 bits 0.0030 instead of 0.0024).  The lowest byte is cut off, not rounded: P is up to
// 2^-15 of itself too small, 1/128 of the half step that dS is rounded by right after.
template <typename T> struct AttnPass;
template <> struct AttnPass<__bf16> {
    static constexpr int PARTS = 3;
    static __device__ __forceinline__ void save(f32x4* at, int lane, const f32x16& p) {
        unsigned d[12];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(p[4 * e + i]);
            d[3 * e] = __builtin_amdgcn_perm(w[1], w[0], 0x05030201u);
            d[3 * e + 1] = __builtin_amdgcn_perm(w[2], w[1], 0x06050302u);
            d[3 * e + 2] = __builtin_amdgcn_perm(w[3], w[2], 0x07060503u);
        }
#pragma unroll
        for (int u = 0; u < 3; ++u)
            at[u * 64 + lane] = (f32x4){__uint_as_float(d[4 * u]), __uint_as_float(d[4 * u + 1]), __uint_as_float(d[4 * u + 2]), __uint_as_float(d[4 * u + 3])};
    }
    f32x4 v[3];
    __device__ __forceinline__ void load(const f32x4* at, int lane) {
#pragma unroll
        for (int u = 0; u < 3; ++u) v[u] = at[u * 64 + lane];
    }
    __device__ __forceinline__ float get(int i) const {
        const int e = i / 4 * 3;
        auto d = [&](int k) { return __float_as_uint(v[(e + k) / 4][(e + k) % 4]); };
        return __uint_as_float(i % 4 == 0 ? __builtin_amdgcn_perm(d(0), d(0), 0x0201000cu) : i % 4 == 1 ? __builtin_amdgcn_perm(d(1), d(0), 0x0504030cu)
                               : i % 4 == 2 ? __builtin_amdgcn_perm(d(2), d(1), 0x0403020cu) : __builtin_amdgcn_perm(d(2), d(2), 0x0302010cu));
    }
};
template <> struct AttnPass<float> {
    static constexpr int PARTS = 4;
    static __device__ __forceinline__ void save(f32x4* at, int lane, const f32x16& p) {
#pragma unroll
        for (int u = 0; u < 4; ++u) at[u * 64 + lane] = (f32x4){p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]};
    }
    f32x4 v[4];
    __device__ __forceinline__ void load(const f32x4* at, int lane) {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = at[u * 64 + lane];
    }
    __device__ __forceinline__ float get(int i) const { return v[i / 4][i % 4]; }
};

template <> struct AttnPass<AttnThree> : AttnPass<float> {};

// X^T (32 of DP x 32 rows) from the rows row0 .. row0 + 31 of a tile, in the row order of AttnProb, and acc += X^T * P
template <typename T, int DP> struct AttnCols;
// one part of bf16 rows, by transposing reads
template <typename L> __device__ __forceinline__ void attn_cols(bf16x8 (&f)[2], const char* tile, int row0, int db, int lane, int part) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const int g = lane >> 4, l = lane & 15;
    const int chunk = (db * 4 + (g & 1) * 2 + ((l & 3) >> 1)) & (L::NCH - 1), low = (l & 1) * 8;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int row = row0 + 16 * u + 4 * (g >> 1) + (l >> 2);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + L::place(row, chunk, part) + low));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + L::place(row + 8, chunk, part) + low));
        f[u] = __builtin_shufflevector(__builtin_bit_cast(bf16x4, a), __builtin_bit_cast(bf16x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
    }
}
template <int DP> struct AttnCols<__bf16, DP> {
    bf16x8 f[2];
    __device__ __forceinline__ void fetch(const char* tile, int row0, int db, int lane) { attn_cols<AttnTile<__bf16, DP>>(f, tile, row0, db, lane, 0); }
    __device__ __forceinline__ void mma(f32x16& acc, const AttnProb<__bf16>& p) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) attn_mma(acc, f[u], p.v[u]);
    }
};
template <int DP> struct AttnCols<AttnThree, DP> {
    bf16x8 f[3][2];
    __device__ __forceinline__ void fetch(const char* tile, int row0, int db, int lane) {
#pragma unroll
        for (int k = 0; k < 3; ++k) attn_cols<AttnTile<AttnThree, DP>>(f[k], tile, row0, db, lane, k);
    }
    __device__ __forceinline__ void mma(f32x16& acc, const AttnProb<AttnThree>& p) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) attn_mma_three(acc, f[0][u], f[1][u], f[2][u], p.v[0][u], p.v[1][u], p.v[2][u]);
    }
};
template <int DP> struct AttnCols<float, DP> {
    typedef AttnTile<float, DP> L;
    float f[16];
    __device__ __forceinline__ void fetch(const char* tile, int row0, int db, int lane) {
        const int col = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            f[i] = *reinterpret_cast<const float*>(tile + L::place(row0 + 8 * (i / 4) + 4 * h + i % 4, (db * 8 + (col >> 2)) & (L::NCH - 1)) + (col & 3) * 4);
    }
    __device__ __forceinline__ void mma(f32x16& acc, const AttnProb<float>& p) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(f[i], p.v[i], acc, 0, 0, 0);
    }
};

// 16 bytes per lane from global memory straight to LDS, lane i at `lds` + 16 i (`lds` the same for the wave); 4 bytes per lane likewise.  No
// registers are held and no LDS writes issued on the way.  The compiler does not see these loads: attn_arrived() waits for them, and it may
// only wait longer for its own loads than it thinks, never shorter.
__device__ __forceinline__ void attn_dma16(void* lds, const void* src) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void attn_dma4(void* lds, const void* src) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void attn_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// waits for all but the last N of a wave's own loads / for its own LDS accesses (a tile that only one wave uses needs no barrier)
template <int N> __device__ __forceinline__ void attn_arrived_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void attn_own_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

static __device__ const f32x4 attn_zeros = {0.f, 0.f, 0.f, 0.f};      // what chunks behind D are loaded from

// A block's share of a tile on its way from global memory to LDS while the previous tile is computed on: straight (VEC), or through registers,
// element by element
// (NT = 64: a wave's own tile)
template <typename T, int DP, int ROWS, int NT, bool VEC> struct AttnStage {
    typedef AttnTile<T, DP> L;
    static constexpr int CNT = (ROWS * L::CPR + NT - 1) / NT;
    typename L::Frag f[VEC ? 1 : CNT];
    static __device__ __forceinline__ int me() { return NT == 64 ? threadIdx.x & 63 : threadIdx.x; }
    static __device__ __forceinline__ bool idle(int c) { return (ROWS * L::CPR) % NT && c >= ROWS * L::CPR; }
    __device__ __forceinline__ void begin(int i, char* tile, const typename L::In* row, int D) {
        const int c = me() + i * NT;
        if (idle(c)) return;
        if (VEC) {
            const int e = L::chunk_at(c) * L::EPC;
            const typename L::In* p = row + e + (L::THREE ? L::part_at(c) * ((D + 7) & ~7) : 0);
            attn_dma16(tile + (c & ~63) * 16, e < D ? (const void*)p : (const void*)&attn_zeros);
        } else {
            f[i] = L::template fetch<false>(row, L::chunk_at(c), D);
        }
    }
    // rows row0 ..: those behind `last` repeat it (their products are masked)
    __device__ __forceinline__ void begin(char* tile, const typename L::In* base, long long ts, int row0, int last, int D) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) begin(i, tile, base + (size_t)min(row0 + (me() + i * NT) / L::CPR, last) * ts, D);
    }
    // packed rows: token r / G, head r % G
    __device__ __forceinline__ void begin_packed(char* tile, const typename L::In* base, long long ts, long long hs, int row0, int last, int G, int D) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int r = min(row0 + (me() + i * NT) / L::CPR, last), t = r / G;
            begin(i, tile, base + (size_t)t * ts + (size_t)(r - t * G) * hs, D);
        }
    }
    __device__ __forceinline__ void finish(char* tile) const {
        if (VEC) return;
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            const int c = me() + i * NT;
            if (!idle(c)) *reinterpret_cast<typename L::Frag*>(tile + c * 16) = f[i];
        }
    }
};

// Element `row` of packed rows (token row / G, head row % G) on its way towards the first row, `step` rows at a time, without a division
template <typename P> struct AttnCursor {
    P* p;
    int head;
    long long back, wrap;      // a step: `step / G` tokens and `step % G` heads back; a head below 0 is G heads on, a token before
    int less, G;
    __device__ __forceinline__ void set(P* base, long long ts, long long hs, int row, int step, int G_) {
        G = G_;
        const int t = row / G;
        head = row - t * G;
        p = base + (long long)t * ts + (long long)head * hs;
        less = step % G;
        back = (long long)(step / G) * ts + (long long)less * hs;
        wrap = (long long)G * hs - ts;
    }
    __device__ __forceinline__ void move() {
        p -= back;
        head -= less;
        if (head < 0) { head += G; p += wrap; }
    }
};

// column `col`'s accumulators acc[DB] (d = 32 db + 8 (i / 4) + 4 h + i % 4) times f into a row of D elements
template <typename T, int DB, int DP = DB * 32> __device__ __forceinline__ void attn_store_row(T* row, const f32x16 (&acc)[DB], float f, int h, int D) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const bool whole = (D & 3) == 0;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (db * 32 + q * 8 >= DP) continue;
            const int d = db * 32 + q * 8 + h * 4;
            T4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (T)(acc[db][4 * q + i] * f);
            if (whole) {
                if (d < D) __builtin_memcpy(__builtin_assume_aligned(row + d, sizeof(T) * 4), &v, sizeof(v));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < D) row[d + i] = v[i];
            }
        }
}

__device__ __forceinline__ float attn_other_half(float x) { return __shfl_xor(x, 32); }

// Infinities and NaN behind the causal edge.  A probability of 0 times one of them is NaN, and on the edge's tiles a product has rows that see
// a key beside rows that do not.  Values of those tiles are looked at (attn_odd), and a wave that finds one makes its sums again, key by key,
// with the keys a row does not see left out: `c`, `m` and `l` stay, the scores were masked before anything was made of them.
template <typename T, int DP> __device__ __forceinline__ bool attn_odd(const char* tile, int row0, int lane) {
    typedef AttnTile<T, DP> L;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < L::NCH / 2; ++i) {
        const typename L::Frag f = L::frag(tile, row0 + (lane & 31), i, lane >> 5);
#pragma unroll
        for (int e = 0; e < L::EPC; ++e) odd |= !(fabsf((float)f[e]) <= 3.4028234664e38f);
    }
    return odd;
}
template <typename T> __device__ __forceinline__ float attn_element(const typename AttnElem<T>::In* row, int d, int D) {
    float x = (float)row[d];
    if (AttnElem<T>::THREE) x += (float)row[((D + 7) & ~7) + d] + (float)row[2 * ((D + 7) & ~7) + d];
    return x;
}
// keys first, first + 1, ... + 31, first + step, ... below `end`
template <typename T, int DP, int DB>
__device__ __forceinline__ void attn_redo(const typename AttnElem<T>::In* q, const typename AttnElem<T>::In* kb, long long k_ts,
                                          const typename AttnElem<T>::In* vb, long long v_ts, f32x16 (&acc)[DB], int D, float c, float m, int limit,
                                          int first, int step, int end, int lane) {
    const int h = lane >> 5;
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = (f32x16)(0.f);
    for (int j0 = first; j0 < end; j0 += step)
        for (int j = j0; j < min(j0 + 32, end); ++j) {
            const typename AttnElem<T>::In *kr = kb + (size_t)j * k_ts, *vr = vb + (size_t)j * v_ts;
            float s = 0.f;
            for (int d = h; d < D; d += 2) s = fmaf(attn_element<T>(q, d, D), attn_element<T>(kr, d, D), s);
            s += attn_other_half(s);
            if (j >= limit) continue;
            const float p = __builtin_amdgcn_exp2f(fmaf(s, c, -ref));
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int d = db * 32 + 8 * (i / 4) + 4 * h + i % 4;
                    if (d < D) acc[db][i] = fmaf(p, attn_element<T>(vr, d, D), acc[db][i]);
                }
        }
}

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

// The running softmax of a wave's 32 rows over tiles of 32 keys: m is a reference for the exponents (see packed_attn.hip)
template <typename T, int DP> struct AttnRun {
    typedef AttnTile<T, DP> L;
    f32x16 acc[L::DB];
    float m, l;
    bool odd;
    __device__ __forceinline__ void reset() {
        odd = false;
#pragma unroll
        for (int db = 0; db < L::DB; ++db) acc[db] = (f32x16)(0.f);
        m = -INFINITY;
        l = 0.f;
    }
    __device__ __forceinline__ void move(float mx) {
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int db = 0; db < L::DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] *= f;
        }
    }
    // keys j0 .. j0 + 31 of which those below `limit` are this lane's row's
    __device__ __forceinline__ void tile(const char* tk, const char* tv, const AttnRows<T, DP>& q, float c, int j0, int limit, bool edge, bool causal,
                                         int lane) {
        const int col = lane & 31, h = lane >> 5;
        AttnRows<T, DP> k;
        k.fetch(tk, col, h);
        attn_fence();
        f32x16 s = attn_product(k, q);
        if (edge) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (j0 + 8 * (i / 4) + 4 * h + i % 4 >= limit) s[i] = -INFINITY;
            if (causal) odd |= attn_odd<T, DP>(tv, 0, lane);
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        move(fmaxf(mx, attn_other_half(mx)) * c);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -ref));
            l += s[i];
        }
        AttnProb<T> p;
        p.set(s);
#pragma unroll
        for (int db = 0; db < L::DB; ++db) {
            AttnCols<T, DP> v;
            v.fetch(tv, 0, db, lane);
            v.mma(acc[db], p);
        }
    }
};
__device__ __forceinline__ float attn_lse(float m, float l) {      // m in powers of two
    return l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f : -INFINITY;
}
__device__ __forceinline__ float attn_inv(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }

// host side (packed_attn.hip)
int attn_geom(AttnGeom& g, const int* off_q, const int* off_k, const int* k_len, float temperature, int causal, int B, int Nq, int Nk, int Hq,
              int Hk, int D, int act);
bool attn_aligned(const AttnTensor* t, int n, int D, int act);
// packed_attn_planes.hip: fp32 inputs laid out as rows [3][D rounded up to 8] of bf16 (see AttnThree)
constexpr int ATTN_MAX_PLANES = 4;
bool attn_three(const AttnGeom& g, int act, bool vec);
long long attn_planes_floats(const AttnGeom& g, long long q_like, long long k_like);
void attn_planes(const AttnGeom& g, const AttnTensor* in, const int* N, const int* H, int n, float* work, AttnTensor* out, hipStream_t stream);
// packed_attn_rows.hip: kernels whose unit is a wave, for few rows per sequence
struct AttnSplit { int waves, chunk, splits; };     // waves that share a task, keys per block, blocks per sequence (1: no partial results)
AttnSplit attn_split(const AttnGeom& g, int max_q, int max_k, int act);
bool attn_short(const AttnGeom& g, int max_q, int max_k);
bool attn_rows_fwd(const AttnGeom& g, const AttnSplit& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, void* out, long long o_ts,
                   long long o_hs, float* lse, float* work, int act, bool vec, hipStream_t stream);
bool attn_short_bwd(const AttnGeom& g, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, const AttnTensor& o, const AttnTensor& go,
                    const float* lse, void* dq, void* dk, void* dv, int act, bool vec, hipStream_t stream);
