// Backward of the attention over packed token sequences (see packed_attn.h for the layout of a product):
//   P = exp(S - lse),  delta = sum(dOut * Out),  dP = dOut V^T,  dS = P (dP - delta) / temperature
//   dQ = dS K,   dV = P^T dOut,   dK = dS^T Q,   dK and dV summed over the query heads of a group
// Two kernels, each recomputing S and dP from the stored lse: one owns rows of queries (dQ, and delta on its way), one owns keys (dK, dV).
// That is 7 products instead of the 5 of a single kernel that would add its share of dQ to memory from every key tile -- but no atomics: the
// result does not depend on the order blocks run in, and no fp32 copy of dQ is written, read back and rounded.  The group's heads are
// consecutive rows of one problem, so dK and dV are sums inside a block as well.
// Bound: the matrix units, and in dK/dV the LDS reads beside them (four operands of 8 KB for every 32 x 32 tile).  Fastest launches: five causal
// sequences of 2832 to 5000 tokens, 16/4 heads of 128, bf16: dQ 533 us (919 TFLOP/s), dK/dV 793 us (823); the clock falls with the power, the
// medians are 5 % above.  Two sequences of 4096 and 1587 tokens, 8 heads of 32, fp32 in three bf16 parts: dQ 190 us, dK/dV 305 (in fp32 products
// 289 and 398).
#include "packed_attn.h"

namespace {

template <typename T, int DP, int NW, int TK, int KSPLIT, bool VEC>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(AttnTile<T, DP>::WAVES))) void packed_attn_dq_kernel(
    const AttnGeom g, const AttnTensor q, const AttnTensor k, const AttnTensor v, const AttnTensor o, const AttnTensor go, const AttnTensor go_raw,
    const float* __restrict__ lse, typename AttnElem<T>::Out* __restrict__ dq, float* __restrict__ rowstat, int slots) {
    typedef AttnTile<T, DP> L;
    typedef typename AttnElem<T>::In In;
    typedef typename AttnElem<T>::Out Out;
    constexpr int NT = NW * 64, GROUPS = NW / KSPLIT, BM = GROUPS * 32, SHIFT = BM == 256 ? 8 : BM == 128 ? 7 : 6;
    __shared__ alignas(16) AttnBuffers<T, DP, TK> lds;
    auto &lds_k = lds.k, &lds_v = lds.v;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    attn_fill_outside<Out>(g.off_q, g.B, g.Nq, dq, (long long)g.Hq * g.D, g.D, g.Hq, g.D, nullptr, blockIdx.x, gridDim.x);
    const int hk = blockIdx.x % g.Hk;
    int b, tile;
    if (g.sorted ? !attn_find_sorted<false>(g, BM, blockIdx.x / g.Hk, b, tile)
                 : !attn_find(g.off_q, g.B, g.Nq, g.G, SHIFT, slots - 1 - (int)(blockIdx.x / g.Hk), b, tile)) return;
    const AttnSeq s = attn_seq(g, b);
    const int rows = s.lq * g.G;
    if (tile * BM >= rows) return;
    const int row0 = tile * BM + wave % GROUPS * 32, share = KSPLIT == 1 ? 0 : wave / GROUPS;      // KSPLIT waves have the same rows and every KSPLIT-th 32 keys
    const int row = min(row0 + col, rows - 1), tok = row / g.G, head = hk * g.G + row - tok * g.G;
    const int shift = s.lk - s.lq;
    auto limit_of = [&](int r) { return g.causal ? min(max(min(r, rows - 1) / g.G + shift + 1, 0), s.lk) : s.lk; };
    const int limit = limit_of(row);
    const int wave_lo = limit_of(row0), wave_hi = row0 < rows ? limit_of(row0 + 31) : 0, block_hi = limit_of(tile * BM + BM - 1);

    AttnRows<T, DP> qf, gf;
    qf.template fetch_global<VEC>((const In*)q.p + (size_t)(s.q0 + tok) * q.ts + (size_t)head * q.hs, h, g.D);
    gf.template fetch_global<VEC>((const In*)go.p + (size_t)(s.q0 + tok) * go.ts + (size_t)head * go.hs, h, g.D);
    float dl;
    {           // delta from dOut and Out as they are stored
        AttnRows<Out, DP> of, gr;
        of.template fetch_global<VEC>((const Out*)o.p + (size_t)(s.q0 + tok) * o.ts + (size_t)head * o.hs, h, g.D);
        gr.template fetch_global<VEC>((const Out*)go_raw.p + (size_t)(s.q0 + tok) * go_raw.ts + (size_t)head * go_raw.hs, h, g.D);
        dl = gr.dot(of);
    }
    dl += attn_other_half(dl);
    const int tiles = (block_hi + TK - 1) / TK;
    const In* kb = (const In*)k.p + (size_t)s.k0 * k.ts + (size_t)hk * k.hs;
    const In* vb = (const In*)v.p + (size_t)s.k0 * v.ts + (size_t)hk * v.hs;
    AttnStage<T, DP, TK, NT, VEC> ks, vs;
    if (tiles) {
        ks.begin(lds_k[0], kb, k.ts, 0, s.lk - 1, g.D);
        vs.begin(lds_v[0], vb, v.ts, 0, s.lk - 1, g.D);
        ks.finish(lds_k[0]);
        vs.finish(lds_v[0]);
    }
    const size_t at = (size_t)(s.q0 + tok) * g.Hq + head;
    // a row that saw nothing has lse = -inf: +inf makes its probabilities 0
    float ls = lse[at] * 1.4426950408889634f;
    if (ls == -INFINITY) ls = INFINITY;
    attn_arrived();
    __syncthreads();
    // bf16: rows of a block with at most two tiles of keys take delta as the sum of P dP instead, in a round before the others.  A rounded Out
    // leaves an error in every dS that few keys do not average away (4 series of up to 100 tokens, causal, dK's error against 64 bits
    // 0.0026; of up to 6, 0.0033; both 0.0024 now; 200 series of up to 100 tokens, 8/4 heads of 64: 23 -> 26 us).
    if (sizeof(Out) == 2 && tiles > 0 && tiles <= 2) {
        if (tiles == 2) {
            ks.begin(lds_k[1], kb, k.ts, TK, s.lk - 1, g.D);
            vs.begin(lds_v[1], vb, v.ts, TK, s.lk - 1, g.D);
            ks.finish(lds_k[1]);
            vs.finish(lds_v[1]);
            attn_arrived();
            __syncthreads();
        }
        dl = 0.f;
        for (int j0 = 0; j0 < wave_hi; j0 += 32) {
            const int t = j0 / TK;
            AttnRows<T, DP> x;
            x.fetch(lds_k[t], j0 - t * TK + col, h);
            const f32x16 sc = attn_product(x, qf);
            x.fetch(lds_v[t], j0 - t * TK + col, h);
            const f32x16 dp = attn_product(x, gf);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                dl += j0 + 8 * (i / 4) + 4 * h + i % 4 < limit ? __builtin_amdgcn_exp2f(fmaf(sc[i], g.c, -ls)) * dp[i] : 0.f;
        }
        dl += attn_other_half(dl);
        __syncthreads();
    }
    if (h == 0 && share == 0 && row0 + col < rows) {          // for the dK/dV kernel: lse in powers of two, and delta behind it
        rowstat[at] = ls;
        rowstat[(size_t)g.Nq * g.Hq + at] = dl;
    }

    f32x16 acc[L::DB];
#pragma unroll
    for (int db = 0; db < L::DB; ++db) acc[db] = (f32x16)(0.f);
    for (int it = 0; it < tiles; ++it) {
        const int j0 = it * TK;
        if (it + 1 < tiles) {
            ks.begin(lds_k[(it + 1) & 1], kb, k.ts, j0 + TK, s.lk - 1, g.D);
            vs.begin(lds_v[(it + 1) & 1], vb, v.ts, j0 + TK, s.lk - 1, g.D);
        }
        if (j0 < wave_hi) {
            const char* tk = lds_k[it & 1];
            const char* tv = lds_v[it & 1];
            const bool edge = j0 + TK > wave_lo;
#pragma unroll
            for (int u = 0; u < TK / 32 / KSPLIT; ++u) {
                const int t = u * KSPLIT + share;
                AttnRows<T, DP> x;
                x.fetch(tk, t * 32 + col, h);
                attn_fence();
                f32x16 sc = attn_product(x, qf);
                x.fetch(tv, t * 32 + col, h);
                attn_fence();
                const f32x16 dp = attn_product(x, gf);
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], g.c, -ls)) * (dp[i] - dl);
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (j0 + t * 32 + 8 * (i / 4) + 4 * h + i % 4 >= limit) sc[i] = 0.f;
                }
                AttnProb<T> p;
                p.set(sc);
#pragma unroll
                for (int db = 0; db < L::DB; ++db) {
                    AttnCols<T, DP> kf;
                    kf.fetch(tk, t * 32, db, lane);
                    kf.mma(acc[db], p);
                }
            }
        }
        if (it + 1 < tiles) {
            ks.finish(lds_k[(it + 1) & 1]);
            vs.finish(lds_v[(it + 1) & 1]);
        }
        attn_arrived();
        __syncthreads();
    }
    if constexpr (KSPLIT == 2) {          // the second wave's sum to the first one, through the tiles nobody needs any more
        float* pass = lds.template join<GROUPS>(wave % GROUPS);
        if (share) {
#pragma unroll
            for (int db = 0; db < L::DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) pass[(db * 16 + i) * 64 + lane] = acc[db][i];
        }
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int db = 0; db < L::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] += pass[(db * 16 + i) * 64 + lane];
    }
    if (row0 + col < rows) attn_store_row<Out, L::DB>(dq + at * g.D, acc, g.scale, h, g.D);
}

// A block owns 32 keys for each of its pairs of waves.  The first wave of a pair holds its keys' K and the sum dV, the second V and dK:
//   first:  S = Q K^T, P = exp2(S c - lse), P to LDS, dV^T += dOut^T P          second, one tile behind:  dP = dOut V^T, dS, dK^T += Q^T dS
// Both make half of the products and hold half of the accumulators (one wave with both needs 470 registers and leaves one wave per SIMD with
// nothing to run beside it); the exponentials of one wave run beside the products of the other.  P crosses in the accumulator layout, lane
// by lane.  Q and dOut tiles rotate through three buffers: the one being filled and those of the two roles.
template <typename T, int DP, int PAIRS, bool VEC>
__global__ __launch_bounds__(PAIRS * 128) __attribute__((amdgpu_waves_per_eu(2))) void packed_attn_dkv_kernel(
    const AttnGeom g, const AttnTensor q, const AttnTensor k, const AttnTensor v, const AttnTensor go, const float* __restrict__ rowstat,
    typename AttnElem<T>::Out* __restrict__ dk, typename AttnElem<T>::Out* __restrict__ dv, int slots) {
    typedef AttnTile<T, DP> L;
    typedef typename AttnElem<T>::In In;
    typedef typename AttnElem<T>::Out Out;
    constexpr int NT = PAIRS * 128, BN = PAIRS * 32, SHIFT = PAIRS == 4 ? 7 : 6, TQ = sizeof(T) == 2 && (PAIRS == 4 || L::RB <= 128) ? 64 : 32;      // AttnThree, fp32: 32
    constexpr bool EARLY = L::RB <= 256;       // registers for the transposed operand beside the first product (not for fp32 rows of 512 bytes)
    __shared__ alignas(16) char lds_q[3][TQ * L::RB], lds_g[3][TQ * L::RB];
    __shared__ f32x4 lds_p[2][PAIRS][TQ / 32][AttnPass<T>::PARTS][64];
    __shared__ alignas(16) float lds_s[3][2][TQ];       // lse in powers of two and delta of a tile's rows
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31, pair = wave % PAIRS;
    const bool second = wave >= PAIRS;
    attn_fill_outside<Out>(g.off_k, g.B, g.Nk, dk, (long long)g.Hk * g.D, g.D, g.Hk, g.D, nullptr, blockIdx.x, gridDim.x);
    attn_fill_outside<Out>(g.off_k, g.B, g.Nk, dv, (long long)g.Hk * g.D, g.D, g.Hk, g.D, nullptr, blockIdx.x, gridDim.x);
    const int hk = blockIdx.x % g.Hk;
    int b, tile;
    // the first keys of a causal sequence are seen by the most rows: they start first
    if (g.sorted ? !attn_find_sorted<true>(g, BN, blockIdx.x / g.Hk, b, tile)
                 : !attn_find(g.off_k, g.B, g.Nk, 1, SHIFT, (int)(blockIdx.x / g.Hk), b, tile)) return;
    const AttnSeq s = attn_seq(g, b);
    if (tile * BN >= s.room) return;
    const int key0 = tile * BN + pair * 32, key = key0 + col;
    const int rows = s.lq * g.G, shift = s.lk - s.lq;
    f32x16 acc[L::DB];
#pragma unroll
    for (int db = 0; db < L::DB; ++db) acc[db] = (f32x16)(0.f);

    // rows [start, rows) see a key of this block; keys behind lk are room in a cache that nothing sees
    int start = g.causal ? min(max(tile * BN - shift, 0), s.lq) * g.G : 0;
    if (tile * BN >= s.lk) start = rows;
    const int tiles = (rows - start + TQ - 1) / TQ;
    if (tiles > 0) {
        AttnRows<T, DP> own;
        {
            const AttnTensor& x = second ? v : k;
            own.template fetch_global<VEC>((const In*)x.p + (size_t)(s.k0 + min(key, s.lk - 1)) * x.ts + (size_t)hk * x.hs, h, g.D);
        }
        const In* qb = (const In*)q.p + (size_t)s.q0 * q.ts + (size_t)hk * g.G * q.hs;
        const In* gb = (const In*)go.p + (size_t)s.q0 * go.ts + (size_t)hk * g.G * go.hs;
        const float* lb = rowstat + (second ? (size_t)g.Nq * g.Hq : 0) + (size_t)s.q0 * g.Hq + hk * g.G;
        // from the last rows to the first: the blocks of a causal sequence then walk over the same rows at the same time, and find them in L2
        auto row_of = [&](int it) { return start + (tiles - 1 - it) * TQ; };
        typedef AttnStage<T, DP, TQ, NT, VEC> Stage;
        Stage qs, gs;
        AttnCursor<const In> cq[Stage::CNT], cg[Stage::CNT];
        AttnCursor<const float> cl;
        // lse (first waves) and delta (second waves) of the tile's rows go to LDS in equal shares
        constexpr int SHARE = TQ / PAIRS;
        const int lrow = pair * SHARE + lane % SHARE;
        const bool lme = lane < SHARE;
        // the first tile repeats the last row behind it, and masks it
#pragma unroll
        for (int i = 0; i < Stage::CNT; ++i) {
            const int r = row_of(0) + min((int)(threadIdx.x + i * NT) / L::CPR, TQ - 1);
            const int t = min(r, rows - 1) / g.G, hd = min(r, rows - 1) - t * g.G;
            qs.begin(i, lds_q[0], qb + (size_t)t * q.ts + (size_t)hd * q.hs, g.D);
            gs.begin(i, lds_g[0], gb + (size_t)t * go.ts + (size_t)hd * go.hs, g.D);
            cq[i].set(qb, q.ts, q.hs, r, TQ, g.G);
            cg[i].set(gb, go.ts, go.hs, r, TQ, g.G);
        }
        {
            const int r = row_of(0) + lrow, t = min(r, rows - 1) / g.G;
            if (lme) attn_dma4(&lds_s[0][second][pair * SHARE], lb + (size_t)t * g.Hq + (min(r, rows - 1) - t * g.G));
            cl.set(lb, g.Hq, 1, r, TQ, g.G);
        }
        auto begin = [&](int buf) {
#pragma unroll
            for (int i = 0; i < Stage::CNT; ++i) {
                cq[i].move();
                cg[i].move();
                qs.begin(i, lds_q[buf], cq[i].p, g.D);
                gs.begin(i, lds_g[buf], cg[i].p, g.D);
            }
            cl.move();
            if (lme) attn_dma4(&lds_s[buf][second][pair * SHARE], cl.p);
        };
        auto finish = [&](int buf) {
            qs.finish(lds_q[buf]);
            gs.finish(lds_g[buf]);
            attn_arrived();
        };
        // causal: a key is seen by the rows from (key - shift) * G on.  Tiles before `seen` have none for this pair's keys, tiles from
        // `whole` on see all of them
        const int first = g.causal ? max(key - shift, 0) * g.G : 0;
        const int seen = key0 >= s.lk ? rows : g.causal ? max(key0 - shift, 0) * g.G : 0, whole = g.causal ? max(key0 + 31 - shift, 0) * g.G : 0;
        finish(0);
        __syncthreads();
        int cur = 0, prev = 2, next = 1;
        for (int it = 0; it <= tiles; ++it) {
            if (it + 1 < tiles) begin(next);
            if (!second) {
                const int r0 = row_of(it);
                if (it < tiles && min(r0 + TQ, rows) > seen) {
#pragma unroll
                    for (int t = 0; t < TQ / 32; ++t) {
                        AttnRows<T, DP> x;
                        x.fetch(lds_q[cur], t * 32 + col, h);
                        attn_fence();
                        f32x16 sc = attn_product(x, own);
                        f32x4 ls[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) ls[e] = *reinterpret_cast<const f32x4*>(&lds_s[cur][0][t * 32 + 8 * e + 4 * h]);
                        AttnCols<T, DP> y[L::DB];
#pragma unroll
                        for (int db = 0; db < L::DB; ++db)
                            if (EARLY) y[db].fetch(lds_g[cur], t * 32, db, lane);
                        attn_fence();
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], g.c, -ls[i / 4][i % 4]));
                        if (r0 < whole || r0 + TQ > rows) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int r = r0 + t * 32 + 8 * (i / 4) + 4 * h + i % 4;
                                if (r < first || r >= rows) sc[i] = 0.f;
                            }
                        }
                        AttnProb<T> p;
                        p.set(sc);
                        AttnPass<T>::save(&lds_p[it & 1][pair][t][0][0], lane, sc);
#pragma unroll
                        for (int db = 0; db < L::DB; ++db) {
                            if (!EARLY) y[db].fetch(lds_g[cur], t * 32, db, lane);
                            y[db].mma(acc[db], p);
                        }
                    }
                }
            } else if (it > 0 && min(row_of(it - 1) + TQ, rows) > seen) {
#pragma unroll
                for (int t = 0; t < TQ / 32; ++t) {
                    AttnRows<T, DP> x;
                    x.fetch(lds_g[prev], t * 32 + col, h);
                    attn_fence();
                    f32x16 dp = attn_product(x, own);
                    f32x4 dl[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) dl[e] = *reinterpret_cast<const f32x4*>(&lds_s[prev][1][t * 32 + 8 * e + 4 * h]);
                    AttnPass<T> p;
                    p.load(&lds_p[(it - 1) & 1][pair][t][0][0], lane);
                    AttnCols<T, DP> y[L::DB];
#pragma unroll
                    for (int db = 0; db < L::DB; ++db)
                        if (EARLY) y[db].fetch(lds_q[prev], t * 32, db, lane);
                    attn_fence();
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] = p.get(i) * (dp[i] - dl[i / 4][i % 4]);
                    AttnProb<T> ds;
                    ds.set(dp);
#pragma unroll
                    for (int db = 0; db < L::DB; ++db) {
                        if (!EARLY) y[db].fetch(lds_q[prev], t * 32, db, lane);
                        y[db].mma(acc[db], ds);
                    }
                }
            }
            if (it + 1 < tiles) finish(next);
            __syncthreads();
            const int t = prev;
            prev = cur;
            cur = next;
            next = t;
        }
    }
    if (key >= s.room) return;
    // a key in the room behind lk: its column repeated the last key's
    if (key >= s.lk)
#pragma unroll
        for (int db = 0; db < L::DB; ++db) acc[db] = (f32x16)(0.f);
    attn_store_row<Out, L::DB>((second ? dk : dv) + ((size_t)(s.k0 + key) * g.Hk + hk) * g.D, acc, second ? g.scale : 1.f, h, g.D);
}

struct Bwd {
    AttnGeom g;
    AttnTensor q, k, v, o, go, go_raw;          // go_raw: dOut as it came, where go is its parts
    const float* lse;
    void *dq, *dk, *dv;
    float* rowstat;
    bool vec;
    hipStream_t stream;
};

template <typename T, int DP, int NW, int TK, int KSPLIT, bool VEC> bool launch_dq(const Bwd& a) {
    constexpr int BM = NW / KSPLIT * 32, SHIFT = BM == 256 ? 8 : BM == 128 ? 7 : 6;
    AttnGeom g = a.g;
    g.sorted = attn_sorts(g, (long long)g.Nq * g.G, BM);
    const int slots = attn_slots((long long)g.Nq * g.G, g.B, SHIFT);
    if (!attn_grid((long long)slots * g.Hk, NW * 64)) return false;
    hipLaunchKernelGGL((packed_attn_dq_kernel<T, DP, NW, TK, KSPLIT, VEC>), dim3(slots * g.Hk), dim3(NW * 64), 0, a.stream, g, a.q, a.k, a.v, a.o, a.go,
                       a.go_raw, a.lse, (typename AttnElem<T>::Out*)a.dq, a.rowstat, slots);
    return true;
}
template <typename T, int DP, int PAIRS, bool VEC> bool launch_dkv(const Bwd& a) {
    AttnGeom g = a.g;
    g.sorted = attn_sorts(g, g.Nk, PAIRS * 32);
    const int slots = attn_slots(g.Nk, g.B, PAIRS == 4 ? 7 : 6);
    if (!attn_grid((long long)slots * g.Hk, PAIRS * 128)) return false;
    hipLaunchKernelGGL((packed_attn_dkv_kernel<T, DP, PAIRS, VEC>), dim3(slots * g.Hk), dim3(PAIRS * 128), 0, a.stream, g, a.q, a.k, a.v, a.go, a.rowstat,
                       (typename AttnElem<T>::Out*)a.dk, (typename AttnElem<T>::Out*)a.dv, slots);
    return true;
}
template <typename T, int DP, int NW, int TK, bool VEC> bool launch_v(const Bwd& a) {
    if (a.g.Nq) {
        constexpr int LOW_NW = AttnElem<T>::THREE ? NW : 2, LOW_TK = AttnElem<T>::THREE ? TK : 32;
        const bool fits = TK == 64 && attn_few_blocks(a.g, NW * 32)         ? launch_dq<T, DP, NW, TK, TK == 64 ? 2 : 1, VEC>(a)
                          : !AttnElem<T>::THREE && attn_low_rows(a.g) ? launch_dq<T, DP, LOW_NW, LOW_TK, 1, VEC>(a)
                                                                      : launch_dq<T, DP, NW, TK, 1, VEC>(a);
        if (!fits) return false;
    }
    if (a.g.Nk) {
        // two pairs per block: as long as two blocks fit a CU's LDS (heads of 128: with tiles of 32 rows, for which long sequences would pay)
        constexpr bool SMALL = AttnTile<T, DP>::RB <= (AttnElem<T>::THREE ? 192 : 128), LOW = !AttnElem<T>::THREE && AttnTile<T, DP>::RB <= 256;
        if (SMALL && ((long long)a.g.Nk / 128 + a.g.B) * a.g.Hk < 1024) return launch_dkv<T, DP, SMALL ? 2 : 4, VEC>(a);
        if (LOW && attn_low_keys(a.g)) return launch_dkv<T, DP, LOW ? 2 : 4, VEC>(a);
        return launch_dkv<T, DP, 4, VEC>(a);
    }
    return true;
}
template <typename T, int DP, int NW, int TK> bool launch(const Bwd& a) {
    return a.vec ? launch_v<T, DP, NW, TK, true>(a) : launch_v<T, DP, NW, TK, AttnElem<T>::THREE>(a);
}

}  // namespace

extern "C" int uncr_packed_attn_bwd_work(int max_q, int max_k, int B, int Nq, int Nk, int Hq, int Hk, int D, int act) {
    AttnGeom g;
    static const int none = 0;
    if (attn_geom(g, &none, &none, nullptr, 1.f, 0, B, Nq, Nk, Hq, Hk, D, act) != UNCR_OK || attn_short(g, max_q, max_k)) return 0;
    return attn_three(g, act, true) ? (int)attn_planes_floats(g, 2, 2) : 0;
}

extern "C" int uncr_packed_attn_bwd(const void* q, long long q_ts, long long q_hs, const void* k, long long k_ts, long long k_hs, const void* v,
                                    long long v_ts, long long v_hs, const void* out, long long o_ts, long long o_hs, const void* dout,
                                    long long do_ts, long long do_hs, const float* lse, void* dq, void* dk, void* dv, float* rowstat,
                                    const int* off_q, const int* off_k, const int* k_len, float temperature, int causal, int max_q,
                                    int max_k, float* work, long long work_floats, int B, int Nq, int Nk, int Hq, int Hk, int D, int act,
                                    hipStream_t stream) {
    Bwd a;
    const int rc = attn_geom(a.g, off_q, off_k, k_len, temperature, causal, B, Nq, Nk, Hq, Hk, D, act);
    if (rc != UNCR_OK) return rc;
    if (Nq && (!q || !out || !dout || !lse || !dq || !rowstat)) return UNCR_EINVAL;
    if (Nk && (!k || !v || !dk || !dv)) return UNCR_EINVAL;
    if ((D & 3) == 0) {         // the epilogue's 4-element stores
        const uintptr_t align = (act ? 2 : 4) * 4;
        if ((uintptr_t)dq % align || (uintptr_t)dk % align || (uintptr_t)dv % align) return UNCR_EINVAL;
    }
    a.q = {q, q_ts, q_hs}; a.k = {k, k_ts, k_hs}; a.v = {v, v_ts, v_hs}; a.o = {out, o_ts, o_hs}; a.go = a.go_raw = {dout, do_ts, do_hs};
    a.lse = lse; a.dq = dq; a.dk = dk; a.dv = dv; a.rowstat = rowstat; a.stream = stream;
    const AttnTensor all[] = {a.q, a.k, a.v, a.o, a.go};
    a.vec = attn_aligned(all, 5, D, act);
    if (Nq == 0 && Nk == 0) return UNCR_OK;
    bool fits;
    if (attn_short(a.g, max_q, max_k)) {
        fits = attn_short_bwd(a.g, a.q, a.k, a.v, a.o, a.go, lse, dq, dk, dv, act, a.vec, stream);
    } else if (attn_three(a.g, act, a.vec)) {
        if (!work || work_floats < attn_planes_floats(a.g, 2, 2)) return UNCR_EINVAL;
        const AttnTensor in[4] = {a.q, a.k, a.v, a.go};
        const int n[4] = {Nq, Nk, Nk, Nq}, h[4] = {Hq, Hk, Hk, Hq};
        AttnTensor p[4];
        attn_planes(a.g, in, n, h, 4, work, p, stream);
        a.q = p[0]; a.k = p[1]; a.v = p[2]; a.go = p[3];
        if (D <= 32) fits = launch<AttnThree, 32, 4, 64>(a);
        else fits = launch<AttnThree, 64, 4, 32>(a);
    } else if (act) {
        if (D <= 32) fits = launch<__bf16, 32, 4, 64>(a);
        else if (D <= 64) fits = launch<__bf16, 64, 4, 64>(a);
        else fits = launch<__bf16, 128, 8, 64>(a);
    } else {
        if (D <= 32) fits = launch<float, 32, 4, 64>(a);
        else if (D <= 64) fits = launch<float, 64, 4, 64>(a);
        else fits = launch<float, 128, 4, 32>(a);
    }
    if (!fits) return UNCR_ESHAPE;
    UNCR_LAUNCH_CHECK();
    return UNCR_OK;
}
