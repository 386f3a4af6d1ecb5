// Attention over packed token sequences where a sequence has few query rows (a token or a handful per series over a cache; the short series
// of single pixels).  The unit is a WAVE with 32 rows (G heads of a group x tokens) and its own tiles of 32 keys in LDS, filled straight
// from global memory while the previous tile is computed on; nothing waits for another wave on the way.
//   cache:  bound by the read of keys and values.  `waves` waves of a block take every waves-th tile of a range of keys and join their sums
//           in LDS; a long cache is cut into ranges of `chunk` keys for blocks of their own, whose unnormalised sums, maxima and sums of
//           exponentials are joined by a second launch.
//   short:  both sides are at most two tiles: each wave has a sequence and head of its own (a block of the kernels in packed_attn.hip
//           would leave three of its four waves without rows), and the backward makes all three gradients in one pass over one tile.
// Measured: 24 caches of 331 to 32768 keys, 32/8 heads of 128, bf16: 396 us for 1.88 GB, 4.7 TB/s where a large copy reaches 4.96 (the kernel
// of packed_attn.hip alone: 1043); one token over 1000 keys, 16/4 heads of 64: 9.6 us in one launch, bound by the loads that wait for each
// other (23 us there).  1500 series of up to 30 dates, 16 heads of 16, fp32: forward 43 us, backward 81 (332 and 930 there); the 272 MB they
// move would take 55, the rest are the vector instructions and products of 32 x 32 tiles that are a quarter full.
#include "packed_attn.h"

namespace {

template <typename T, int DP, int NW, bool SHARE, bool VEC>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(SHARE ? 1 : DP * sizeof(T) <= 64 ? 4 : DP <= 32 ? 3 : 2))) void packed_attn_rows_kernel(
    const AttnGeom g, const AttnTensor q, const AttnTensor k, const AttnTensor v, T* __restrict__ out, long long o_ts, long long o_hs,
    float* __restrict__ lse, float* __restrict__ work, int chunk, int splits, int tasks) {
    typedef AttnTile<T, DP> L;
    typedef typename AttnElem<T>::In In;
    typedef typename AttnElem<T>::Out Out;
    typedef AttnStage<T, DP, 32, 64, VEC> Stage;
    constexpr int NBUF = SHARE ? 2 : 1, TILE = 32 * L::RB;
    __shared__ alignas(16) char lds[NW][NBUF][2][TILE];
    __shared__ float lds_m[NW][32], lds_l[NW][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    if (g.fill) attn_fill_outside<Out>(g.off_q, g.B, g.Nq, out, o_ts, o_hs, g.Hq, g.D, lse, blockIdx.x, gridDim.x);
    const int task = SHARE ? blockIdx.x : blockIdx.x * NW + wave;
    if (task >= tasks) return;
    const int hk = task % g.Hk, split = SHARE ? task / g.Hk % splits : 0, slot = SHARE ? task / g.Hk / splits : task / g.Hk;
    int b = slot, part = 0;
    if (SHARE && !attn_find(g.off_q, g.B, g.Nq, g.G, 5, slot, b, part)) return;
    const AttnSeq s = attn_seq(g, b);
    const int rows = s.lq * g.G;
    // one tile of rows with shared waves, all of its sequence's for a wave of its own
    for (int row0 = part * 32; row0 < rows; row0 += 32) {
        const int row = min(row0 + col, rows - 1), tok = row / g.G, head = hk * g.G + row - tok * g.G;
        const int shift = s.lk - s.lq;
        auto limit_of = [&](int r) { return g.causal ? min(max(min(r, rows - 1) / g.G + shift + 1, 0), s.lk) : s.lk; };
        const int limit = limit_of(row), lo = limit_of(row0), hi = limit_of(row0 + 31);
        // this block's keys: ranges of `chunk`, longer ones if `splits` of those do not reach the end
        const int range = SHARE ? max(chunk, ((s.lk + splits - 1) / splits + 31) & ~31) : s.lk;
        const int begin = split * range, end = min(hi, begin + range);

        AttnRows<T, DP> qf;
        qf.template fetch_global<VEC>((const In*)q.p + (size_t)(s.q0 + tok) * q.ts + (size_t)head * q.hs, h, g.D);
        AttnRun<T, DP> run;
        run.reset();
        const In* kb = (const In*)k.p + (size_t)s.k0 * k.ts + (size_t)hk * k.hs;
        const In* vb = (const In*)v.p + (size_t)s.k0 * v.ts + (size_t)hk * v.hs;
        Stage ks, vs;
        constexpr int STEP = SHARE ? NW * 32 : 32;
        int j0 = begin + (SHARE ? wave * 32 : 0), buf = 0;
        if (j0 < end) {
            ks.begin(lds[wave][0][0], kb, k.ts, j0, s.lk - 1, g.D);
            vs.begin(lds[wave][0][1], vb, v.ts, j0, s.lk - 1, g.D);
            ks.finish(lds[wave][0][0]);
            vs.finish(lds[wave][0][1]);
        }
        for (; j0 < end; j0 += STEP) {
            const bool more = j0 + STEP < end;
            if (NBUF == 2 && more) {
                attn_own_lds();
                ks.begin(lds[wave][buf ^ 1][0], kb, k.ts, j0 + STEP, s.lk - 1, g.D);
                vs.begin(lds[wave][buf ^ 1][1], vb, v.ts, j0 + STEP, s.lk - 1, g.D);
                attn_arrived_but<VEC ? 2 * Stage::CNT : 0>();
            } else {
                attn_arrived();
            }
            attn_own_lds();
            run.tile(lds[wave][buf][0], lds[wave][buf][1], qf, g.c, j0, limit, j0 + 32 > lo, g.causal != 0, lane);
            if (more) {
                attn_own_lds();
                if (NBUF == 1) {
                    ks.begin(lds[wave][0][0], kb, k.ts, j0 + STEP, s.lk - 1, g.D);
                    vs.begin(lds[wave][0][1], vb, v.ts, j0 + STEP, s.lk - 1, g.D);
                }
                ks.finish(lds[wave][NBUF == 2 ? buf ^ 1 : 0][0]);
                vs.finish(lds[wave][NBUF == 2 ? buf ^ 1 : 0][1]);
            }
            if (NBUF == 2) buf ^= 1;
        }
        float l = run.l + attn_other_half(run.l), m = run.m;
        if (__any(run.odd))
            attn_redo<T, DP>((const In*)q.p + (size_t)(s.q0 + tok) * q.ts + (size_t)head * q.hs, kb, k.ts, vb, v.ts, run.acc, g.D, g.c, m, limit,
                             begin + (SHARE ? wave * 32 : 0), STEP, end, lane);
        if (!SHARE) {
            if (row0 + col < rows) {
                attn_store_row<Out, L::DB, DP>(out + (size_t)(s.q0 + tok) * o_ts + (size_t)head * o_hs, run.acc, attn_inv(l), h, g.D);
                if (lse && h == 0) lse[(size_t)(s.q0 + tok) * g.Hq + head] = attn_lse(m, l);
            }
            attn_own_lds();
            continue;
        }
        // the waves' sums, brought to one reference and added in LDS: [wave][row][DP] over the tiles, which no wave needs any more
        if (h == 0) {
            lds_m[wave][col] = m;
            lds_l[wave][col] = l;
        }
        __syncthreads();
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, lds_m[w][col]);
        const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < NW; ++w) ll += lds_l[w][col] * __builtin_amdgcn_exp2f(lds_m[w][col] - ref);
        const float f = __builtin_amdgcn_exp2f(m - ref);
        const int live = min(rows - row0, 32);
        constexpr int WB = NBUF * 2 * TILE / 4, ROWS = WB / DP < 32 ? WB / DP : 32;       // floats of a wave's tiles; rows of DP they hold
        float* mine = (float*)&lds[wave][0][0][0];
        for (int r0 = 0; r0 < live; r0 += ROWS) {
            if (r0) __syncthreads();
            if (col >= r0 && col < r0 + ROWS && col < live) {
#pragma unroll
                for (int db = 0; db < L::DB; ++db)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = db * 32 + 8 * e + 4 * h;
                        if (d < DP)
                            *reinterpret_cast<f32x4*>(mine + (col - r0) * DP + d) =
                                (f32x4){run.acc[db][4 * e] * f, run.acc[db][4 * e + 1] * f, run.acc[db][4 * e + 2] * f, run.acc[db][4 * e + 3] * f};
                    }
            }
            __syncthreads();
            const int n = min(live - r0, ROWS);
            for (int i = threadIdx.x; i < n * DP; i += NW * 64) {
                const int r = i / DP, d = i % DP;
                if (d >= g.D) continue;
                float a = 0.f, lr = 0.f, mr = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    a += *((const float*)&lds[w][0][0][0] + i);
                    mr = fmaxf(mr, lds_m[w][r0 + r]);
                }
                const int rr = row0 + r0 + r, t = rr / g.G;
                const size_t at = (size_t)(s.q0 + t) * g.Hq + hk * g.G + rr - t * g.G;
                if (splits > 1) {
                    if (mr != -INFINITY) work[((size_t)split * g.Nq * g.Hq + at) * g.D + d] = a;
                } else {
                    const float rf = mr == -INFINITY ? 0.f : mr;
#pragma unroll
                    for (int w = 0; w < NW; ++w) lr += lds_l[w][r0 + r] * __builtin_amdgcn_exp2f(lds_m[w][r0 + r] - rf);
                    out[(size_t)(s.q0 + t) * o_ts + (size_t)(hk * g.G + rr - t * g.G) * o_hs + d] = (T)(a * attn_inv(lr));
                }
            }
        }
        if (wave == 0 && h == 0 && col < live) {
            const size_t at = (size_t)(s.q0 + tok) * g.Hq + head;
            if (splits > 1) {
                float* ml = work + (size_t)splits * g.Nq * g.Hq * g.D + ((size_t)split * g.Nq * g.Hq + at) * 2;
                ml[0] = mm;
                ml[1] = ll;
            } else if (lse) {
                lse[at] = attn_lse(mm, ll);
            }
        }
        return;
    }
}

// out = sum over the splits of exp2(m - max m) (their sums), over the same sum of their l: one wave per row, the sums of 16 splits under way
// at a time
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(const AttnGeom g, const float* __restrict__ work, int splits, T* __restrict__ out,
                                                               long long o_ts, long long o_hs, float* __restrict__ lse) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long at = (long long)blockIdx.x * 4 + wave;
    if (at >= (long long)g.Nq * g.Hq) return;
    const size_t rows = (size_t)g.Nq * g.Hq;
    const float* ml = work + (size_t)splits * rows * g.D;
    const float* row = work + at * g.D;
    const float m = lane < splits ? ml[((size_t)lane * rows + at) * 2] : -INFINITY;
    float l = lane < splits ? ml[((size_t)lane * rows + at) * 2 + 1] : 0.f;
    float x[16][2];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[i][e] = i0 + i < splits && lane + 64 * e < g.D ? row[(size_t)(i0 + i) * rows * g.D + lane + 64 * e] : 0.f;
    };
    fetch(0);
    // is the row one of a sequence's?
    const int tok = (int)(at / g.Hq), head = (int)(at % g.Hq);
    int lo = 0, n = g.B;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool in = lane * step < n && g.off_q[lo + lane * step] <= tok;
        const int cnt = max(__popcll(__ballot(in)), 1);
        lo += (cnt - 1) * step;
        n = min(step, n - (cnt - 1) * step);
    }
    const int q0 = min(max(g.off_q[lo], 0), g.Nq);
    if (tok < q0 || tok >= min(max(g.off_q[lo + 1], q0), g.Nq)) return;
    float mm = m;
#pragma unroll
    for (int d = 32; d; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
    float f = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
    if (m != m) f = m;                              // NaN sums stay NaN, also those of a row that has no maximum because all its scores are NaN
    l = m == -INFINITY && l == l ? 0.f : l * f;
#pragma unroll
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    float a[2] = {0.f, 0.f};
    for (int i0 = 0; i0 < splits; i0 += 16) {
        if (i0) fetch(i0);
#pragma unroll
        for (int i = 0; i < 16; ++i) {              // a split without keys has left its row unwritten: f = 0
            const float fi = i0 + i < splits ? __shfl(f, i0 + i) : 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) a[e] += fi == 0.f ? 0.f : x[i][e] * fi;
        }
    }
    const float inv = attn_inv(l);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < g.D) out[(size_t)tok * o_ts + (size_t)head * o_hs + lane + 64 * e] = (T)(a[e] * inv);
    if (lse && lane == 0) lse[at] = attn_lse(mm, l);
}

// All gradients of short sequences, a wave per sequence and key head.  One tile of keys: P and dS are made once per tile of rows (columns:
// rows), give dQ as they are, and cross a 32 x 32 patch of LDS to become columns of keys for dK and dV.  More keys than a tile: the same for
// every tile of keys, and dQ in a second round.
// delta is not taken from Out but is the sum of P dP, which one tile of keys has at hand (so Out is not read) and for which bf16 storage makes
// a round before the others: a rounded Out leaves an error in every dS that rows with few keys do not average away (series of up to 6 dates,
// dQ's error against 64 bits 0.0031; up to 64 dates 0.0027; both 0.0024 now, what the rounding of dS and of the result make up; the round costs
// 90 -> 98 us with 1500 series of up to 64 dates, 8 heads of 32).
template <typename T, int DP, int NW, bool VEC>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DP <= 32 ? 3 : 2))) void packed_attn_short_bwd_kernel(
    const AttnGeom g, const AttnTensor q, const AttnTensor k, const AttnTensor v, const AttnTensor o, const AttnTensor go,
    const float* __restrict__ lse, T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv) {
    typedef AttnTile<T, DP> L;
    typedef typename AttnElem<T>::In In;
    typedef typename AttnElem<T>::Out Out;
    typedef AttnStage<T, DP, 32, 64, VEC> Stage;
    constexpr int TILE = 32 * L::RB, PS = 36;
    __shared__ alignas(16) char lds[NW][4][TILE];
    __shared__ alignas(16) float patch[NW][32 * PS];
    __shared__ float lds_d[sizeof(T) == 2 ? NW : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    attn_fill_outside<Out>(g.off_q, g.B, g.Nq, dq, (long long)g.Hq * g.D, g.D, g.Hq, g.D, nullptr, blockIdx.x, gridDim.x);
    attn_fill_outside<Out>(g.off_k, g.B, g.Nk, dk, (long long)g.Hk * g.D, g.D, g.Hk, g.D, nullptr, blockIdx.x, gridDim.x);
    attn_fill_outside<Out>(g.off_k, g.B, g.Nk, dv, (long long)g.Hk * g.D, g.D, g.Hk, g.D, nullptr, blockIdx.x, gridDim.x);
    const int task = blockIdx.x * NW + wave, b = task / g.Hk, hk = task - b * g.Hk;
    if (b >= g.B) return;
    const AttnSeq s = attn_seq(g, b);
    const int rows = s.lq * g.G, shift = s.lk - s.lq;
    char *tk = lds[wave][0], *tv = lds[wave][1], *tq = lds[wave][2], *tg = lds[wave][3];
    float* pt = patch[wave];
    const In* kb = (const In*)k.p + (size_t)s.k0 * k.ts + (size_t)hk * k.hs;
    const In* vb = (const In*)v.p + (size_t)s.k0 * v.ts + (size_t)hk * v.hs;
    const In* qb = (const In*)q.p + (size_t)s.q0 * q.ts + (size_t)hk * g.G * q.hs;
    const In* gb = (const In*)go.p + (size_t)s.q0 * go.ts + (size_t)hk * g.G * go.hs;
    Stage s0, s1;
    const bool single = s.lk <= 32, round = !single && sizeof(T) == 2 && rows <= 64;
    bool summed = false;
    auto load_keys = [&](int j0) {
        attn_own_lds();
        s0.begin(tk, kb, k.ts, j0, s.lk - 1, g.D);
        s1.begin(tv, vb, v.ts, j0, s.lk - 1, g.D);
        s0.finish(tk);
        s1.finish(tv);
    };
    float ls = INFINITY, dl = 0.f;
    size_t at = 0;
    auto load_rows = [&](int r0) {
        attn_own_lds();
        s0.begin_packed(tq, qb, q.ts, q.hs, r0, rows - 1, g.G, g.D);
        s1.begin_packed(tg, gb, go.ts, go.hs, r0, rows - 1, g.G, g.D);
        const int row = min(r0 + col, rows - 1), t = row / g.G, hd = hk * g.G + row - t * g.G;
        at = (size_t)(s.q0 + t) * g.Hq + hd;
        ls = lse[at] * 1.4426950408889634f;
        if (ls == -INFINITY || r0 + col >= rows) ls = INFINITY;      // a row that saw nothing, a row behind the last: no probabilities
        s0.finish(tq);
        s1.finish(tg);
        attn_arrived();
        attn_own_lds();
        if (summed) {
            dl = lds_d[sizeof(T) == 2 ? wave : 0][(r0 + col) & 63];
        } else if (!single && !round) {
            AttnRows<T, DP> of, gf;
            of.template fetch_global<VEC>((const In*)o.p + (size_t)(s.q0 + t) * o.ts + (size_t)hd * o.hs, h, g.D);
            gf.fetch(tg, col, h);
            dl = gf.dot(of);
            dl += attn_other_half(dl);
        }
    };
    f32x16 p, ds;
    // P and dP, both 0 where a row does not see a key, and this half's sum of their product
    auto probs = [&](int r0, int j0) {
        AttnRows<T, DP> x, y;
        x.fetch(tk, col, h);
        y.fetch(tq, col, h);
        p = attn_product(x, y);
        x.fetch(tv, col, h);
        y.fetch(tg, col, h);
        ds = attn_product(x, y);
        const int row = min(r0 + col, rows - 1), limit = g.causal ? min(row / g.G + shift + 1, s.lk) : s.lk;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool in = j0 + 8 * (i / 4) + 4 * h + i % 4 < limit && r0 + col < rows;
            p[i] = in ? __builtin_amdgcn_exp2f(fmaf(p[i], g.c, -ls)) : 0.f;
            ds[i] = in ? ds[i] : 0.f;
        }
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) d = fmaf(p[i], ds[i], d);
        return d;
    };
    auto scores = [&](int r0, int j0) {
        const float d = probs(r0, j0);
        if (single) dl = d + attn_other_half(d);
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] = p[i] * (ds[i] - dl);
    };
    auto turn = [&](f32x16& x) {          // columns: rows -> columns: keys
        attn_own_lds();
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4*>(pt + col * PS + 8 * e + 4 * h) = (f32x4){x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
        attn_own_lds();
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = pt[(8 * (i / 4) + 4 * h + i % 4) * PS + col];
    };
    auto add_dq = [&](f32x16 (&a)[L::DB]) {
        AttnProb<T> w;
        w.set(ds);
#pragma unroll
        for (int db = 0; db < L::DB; ++db) {
            AttnCols<T, DP> x;
            x.fetch(tk, 0, db, lane);
            x.mma(a[db], w);
        }
    };
    auto store_dq = [&](int r0, const f32x16 (&a)[L::DB]) {
        if (r0 + col < rows) attn_store_row<Out, L::DB, DP>(dq + at * g.D, a, g.scale, h, g.D);
    };
    if (round) {
        for (int r0 = 0; r0 < rows; r0 += 32) {
            load_rows(r0);
            float d = 0.f;
            for (int j0 = 0; j0 < s.lk; j0 += 32) {
                load_keys(j0);
                attn_arrived();
                attn_own_lds();
                d += probs(r0, j0);
            }
            d += attn_other_half(d);
            if (h == 0) lds_d[sizeof(T) == 2 ? wave : 0][r0 + col] = d;
        }
        attn_own_lds();
        summed = true;
    }
    for (int j0 = 0; j0 < s.room; j0 += 32) {
        f32x16 ak[L::DB], av[L::DB];
#pragma unroll
        for (int db = 0; db < L::DB; ++db) ak[db] = av[db] = (f32x16)(0.f);
        if (j0 < s.lk && rows) {
            load_keys(j0);
            for (int r0 = 0; r0 < rows; r0 += 32) {
                load_rows(r0);
                scores(r0, j0);
                if (single) {
                    f32x16 aq[L::DB];
#pragma unroll
                    for (int db = 0; db < L::DB; ++db) aq[db] = (f32x16)(0.f);
                    add_dq(aq);
                    store_dq(r0, aq);
                }
                AttnProb<T> w;
                turn(p);
                w.set(p);
#pragma unroll
                for (int db = 0; db < L::DB; ++db) {
                    AttnCols<T, DP> x;
                    x.fetch(tg, 0, db, lane);
                    x.mma(av[db], w);
                }
                turn(ds);
                w.set(ds);
#pragma unroll
                for (int db = 0; db < L::DB; ++db) {
                    AttnCols<T, DP> x;
                    x.fetch(tq, 0, db, lane);
                    x.mma(ak[db], w);
                }
            }
        }
        if (j0 + col < s.room) {
            if (j0 + col >= s.lk)
#pragma unroll
                for (int db = 0; db < L::DB; ++db) ak[db] = av[db] = (f32x16)(0.f);
            const size_t ka = ((size_t)(s.k0 + j0 + col) * g.Hk + hk) * g.D;
            attn_store_row<Out, L::DB, DP>(dk + ka, ak, g.scale, h, g.D);
            attn_store_row<Out, L::DB, DP>(dv + ka, av, 1.f, h, g.D);
        }
    }
    if (single && s.lk > 0) return;
    for (int r0 = 0; r0 < rows; r0 += 32) {
        f32x16 aq[L::DB];
#pragma unroll
        for (int db = 0; db < L::DB; ++db) aq[db] = (f32x16)(0.f);
        load_rows(r0);
        for (int j0 = 0; j0 < s.lk; j0 += 32) {
            load_keys(j0);
            attn_arrived();
            attn_own_lds();
            scores(r0, j0);
            add_dq(aq);
        }
        store_dq(r0, aq);
    }
}

struct Rows {
    AttnGeom g;
    AttnSplit s;
    AttnTensor q, k, v;
    void* out;
    long long o_ts, o_hs;
    float *lse, *work;
    hipStream_t stream;
};

template <typename T, int DP, int NW, bool SHARE, bool VEC> bool launch(const Rows& a) {
    const int tasks = SHARE ? attn_slots((long long)a.g.Nq * a.g.G, a.g.B, 5) * a.g.Hk * a.s.splits : a.g.B * a.g.Hk;
    const long long blocks = SHARE ? tasks : ((long long)tasks + NW - 1) / NW;
    if (!attn_grid(blocks, NW * 64)) return false;
    hipLaunchKernelGGL((packed_attn_rows_kernel<T, DP, NW, SHARE, VEC>), dim3((unsigned)blocks), dim3(NW * 64), 0, a.stream, a.g, a.q,
                       a.k, a.v, (T*)a.out, a.o_ts, a.o_hs, a.lse, a.work, a.s.chunk, a.s.splits, tasks);
    if (SHARE && a.s.splits > 1)
        hipLaunchKernelGGL((packed_attn_join_kernel<T>), dim3((unsigned)(((long long)a.g.Nq * a.g.Hq + 3) / 4)), dim3(256), 0, a.stream, a.g, a.work,
                           a.s.splits, (T*)a.out, a.o_ts, a.o_hs, a.lse);
    return true;
}
template <typename T, int DP, bool VEC> bool launch_n(const Rows& a) {
    constexpr int NW = DP * sizeof(T) <= 128 ? 8 : DP * sizeof(T) <= 256 ? 4 : 2;      // a wave's four tiles are 128 rows: 128 KB of LDS per block
    if (DP == 128 || a.s.waves > 1) return launch<T, DP, NW, true, VEC>(a);
    return launch<T, DP < 128 ? DP : 64, 4, false, VEC>(a);           // attn_short: heads up to 64
}
template <typename T, bool VEC> bool launch_d(const Rows& a) {
    return a.g.D <= 16 ? launch_n<T, 16, VEC>(a) : a.g.D <= 32 ? launch_n<T, 32, VEC>(a) : a.g.D <= 64 ? launch_n<T, 64, VEC>(a) : launch_n<T, 128, VEC>(a);
}

struct Short {
    AttnGeom g;
    AttnTensor q, k, v, o, go;
    const float* lse;
    void *dq, *dk, *dv;
    hipStream_t stream;
};
template <typename T, int DP, bool VEC> bool launch_short(const Short& a) {
    const long long blocks = ((long long)a.g.B * a.g.Hk + 3) / 4;
    if (!attn_grid(blocks, 256)) return false;
    hipLaunchKernelGGL((packed_attn_short_bwd_kernel<T, DP, 4, VEC>), dim3((unsigned)blocks), dim3(256), 0, a.stream, a.g, a.q, a.k, a.v, a.o, a.go,
                       a.lse, (T*)a.dq, (T*)a.dk, (T*)a.dv);
    return true;
}
template <typename T, bool VEC> bool launch_short_d(const Short& a) {
    return a.g.D <= 16 ? launch_short<T, 16, VEC>(a) : a.g.D <= 32 ? launch_short<T, 32, VEC>(a) : launch_short<T, 64, VEC>(a);
}

}  // namespace

// Sequences of at most 64 rows and 64 keys by the caller's word (a wrong word costs time, not results), of heads up to 64
bool attn_short(const AttnGeom& g, int max_q, int max_k) {
    return max_q > 0 && max_k > 0 && (long long)max_q * g.G <= 64 && max_k <= 64 && g.D <= 64;
}

// Who shares a task.  Up to 32 rows per sequence (by the caller's word, else on average) are one wave's rows; more go to the kernels of
// packed_attn.hip, which read a key tile once for 128 or 256 rows and have no ranges.  Both sides, 16/4 heads of 128, bf16, packed_attn.hip against these
// tiles of 32 rows with ranges: 64 caches of 2048 keys, 9 tokens each 111 against 153 us, 64 tokens 193 against 332; 24 of 32768, 64 tokens 949
// against 1737.  Few blocks over long caches lose by the rule: 9 tokens over one cache of 32768 keys 692 against 50 us, over 24 of them 918 against
// 503; one token, 64 heads on one key head of 64, one cache of 32768: 434 against 27.
// Without ranges (splits = 1) up to 8 tiles per wave; then ranges of 4096 keys, shorter ones while the launch
// has fewer than eight blocks per CU (caches are filled to different lengths), down to a tile per wave.
AttnSplit attn_split(const AttnGeom& g, int max_q, int max_k, int act) {
    AttnSplit s = {0, 0, 1};
    const long long rows = (long long)(max_q > 0 ? max_q : (g.Nq + g.B - 1) / g.B) * g.G;
    const long long keys = max_k > 0 ? (max_k < g.Nk ? max_k : g.Nk) : (g.Nk + g.B - 1) / g.B;
    if (attn_short(g, max_q, max_k)) { s.waves = 1; return s; }
    if (rows > 32) return s;
    const int dp = g.D <= 16 ? 16 : g.D <= 32 ? 32 : g.D <= 64 ? 64 : 128, bytes = dp * (act ? 2 : 4);
    s.waves = bytes <= 128 ? 8 : bytes <= 256 ? 4 : 2;
    const long long tasks = attn_slots((long long)g.Nq * g.G, g.B, 5) * (long long)g.Hk;
    if (dp < 128 && !attn_grid(tasks, s.waves * 64)) s.waves = 1;         // millions of them: a wave each is what a launch can hold
    if (s.waves == 1 || keys <= 32ll * 8 * s.waves) return s;
    int chunk = 4096;
    while (chunk > 32 * s.waves && tasks * ((keys + chunk - 1) / chunk) < 2048) chunk >>= 1;
    long long n = (keys + chunk - 1) / chunk;
    if (n > 64) n = 64;
    // partial results of a launch are kept under 2^28 floats
    while (n > 1 && (n * g.Nq * g.Hq * (g.D + 2) > (1ll << 28) || n * tasks > (1ll << 30))) n >>= 1;
    s.chunk = (int)(((keys + n - 1) / n + 31) / 32 * 32);
    s.splits = (int)n;
    return s;
}

bool attn_rows_fwd(const AttnGeom& g, const AttnSplit& s, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, void* out, long long o_ts,
                   long long o_hs, float* lse, float* work, int act, bool vec, hipStream_t stream) {
    const Rows a = {g, s, q, k, v, out, o_ts, o_hs, lse, work, stream};
    if (act) return vec ? launch_d<__bf16, true>(a) : launch_d<__bf16, false>(a);
    return vec ? launch_d<float, true>(a) : launch_d<float, false>(a);
}

bool attn_short_bwd(const AttnGeom& g, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, const AttnTensor& o, const AttnTensor& go,
                    const float* lse, void* dq, void* dk, void* dv, int act, bool vec, hipStream_t stream) {
    const Short a = {g, q, k, v, o, go, lse, dq, dk, dv, stream};
    if (act) return vec ? launch_short_d<__bf16, true>(a) : launch_short_d<__bf16, false>(a);
    return vec ? launch_short_d<float, true>(a) : launch_short_d<float, false>(a);
}
