// Forward of the attention over packed token sequences (see packed_attn.h for the layout of a product):
//   S = Q K^T / temperature over the keys a row may see (its own sequence; causal: key j <= i + Lk - Lq),  out = softmax(S) V
// One pass over the keys with the running maximum m and sum l of each row, in fp32 and in powers of two.  m is only a reference for the
// exponents: it is moved -- and out, l rescaled -- when a tile's maximum passes it by more than 8, so the accumulators are rarely touched
// and exponentials stay below 2^8.  Rows that see nothing: out = 0, lse = -inf.
// Bound: the matrix units under the power cap.  A block of 256 rows (8 waves, two per SIMD) reads each tile of 64 keys once for all of them,
// through two buffers, one being filled while the other is used.  Three causal sequences of 16384, 9004 and 15233 tokens, 32/8 heads of 128,
// bf16: 4.77 ms, 1.0 PFLOP/s -- the library's largest bf16 product reaches 1.2 on the same card.  The products of the next tile put between
// the exponentials of this one by hand took 9 % fewer cycles and not less time (the clock falls with the power), so the loop is the plain
// one.  fp32: two sequences of 4096 and 1587 tokens, 8 heads of 32: 254 us in fp32 products, 225 with blocks of half as many rows, 160 in
// three bf16 parts (AttnThree) behind an 8 us launch that takes them apart.
#include "packed_attn.h"

namespace {

template <typename T, int DP, int NW, int TK, int KSPLIT, bool VEC>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(AttnTile<T, DP>::WAVES))) void packed_attn_fwd_kernel(
    const AttnGeom g, const AttnTensor q, const AttnTensor k, const AttnTensor v, typename AttnElem<T>::Out* __restrict__ out, long long o_ts,
    long long o_hs, float* __restrict__ lse, int slots) {
    typedef AttnTile<T, DP> L;
    typedef typename AttnElem<T>::In In;
    typedef typename AttnElem<T>::Out Out;
    constexpr int NT = NW * 64, GROUPS = NW / KSPLIT, BM = GROUPS * 32, SHIFT = BM == 256 ? 8 : BM == 128 ? 7 : 6;
    __shared__ alignas(16) AttnBuffers<T, DP, TK> lds;
    auto &lds_k = lds.k, &lds_v = lds.v;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    if (g.fill) attn_fill_outside<Out>(g.off_q, g.B, g.Nq, out, o_ts, o_hs, g.Hq, g.D, lse, blockIdx.x, gridDim.x);
    const int hk = blockIdx.x % g.Hk;
    int b, tile;
    // the last tiles of a causal sequence are the longest: they start first
    if (g.sorted ? !attn_find_sorted<false>(g, BM, blockIdx.x / g.Hk, b, tile)
                 : !attn_find(g.off_q, g.B, g.Nq, g.G, SHIFT, slots - 1 - (int)(blockIdx.x / g.Hk), b, tile)) return;
    const AttnSeq s = attn_seq(g, b);
    const int rows = s.lq * g.G;
    if (tile * BM >= rows) return;
    const int row0 = tile * BM + wave % GROUPS * 32, share = KSPLIT == 1 ? 0 : wave / GROUPS;      // KSPLIT waves have the same rows and every KSPLIT-th 32 keys
    const int row = min(row0 + col, rows - 1), tok = row / g.G, head = hk * g.G + row - tok * g.G;
    // keys [0, limit) are visible to this lane's row
    const int shift = s.lk - s.lq;
    auto limit_of = [&](int r) { return g.causal ? min(max(min(r, rows - 1) / g.G + shift + 1, 0), s.lk) : s.lk; };
    const int limit = limit_of(row);
    const int wave_lo = limit_of(row0), wave_hi = row0 < rows ? limit_of(row0 + 31) : 0, block_hi = limit_of(tile * BM + BM - 1);

    AttnRows<T, DP> qf;
    qf.template fetch_global<VEC>((const In*)q.p + (size_t)(s.q0 + tok) * q.ts + (size_t)head * q.hs, h, g.D);
    f32x16 acc[L::DB];
#pragma unroll
    for (int db = 0; db < L::DB; ++db) acc[db] = (f32x16)(0.f);
    float m = -INFINITY, l = 0.f;
    bool odd = false;

    const In* kb = (const In*)k.p + (size_t)s.k0 * k.ts + (size_t)hk * k.hs;
    const In* vb = (const In*)v.p + (size_t)s.k0 * v.ts + (size_t)hk * v.hs;
    constexpr int SUB = TK / 32 / KSPLIT;
    const int tiles = (block_hi + TK - 1) / TK;
    AttnStage<T, DP, TK, NT, VEC> ks, vs;
    if (tiles) {
        ks.begin(lds_k[0], kb, k.ts, 0, s.lk - 1, g.D);
        vs.begin(lds_v[0], vb, v.ts, 0, s.lk - 1, g.D);
        ks.finish(lds_k[0]);
        vs.finish(lds_v[0]);
    }
    attn_arrived();
    __syncthreads();
    for (int it = 0; it < tiles; ++it) {
        const int j0 = it * TK;
        if (it + 1 < tiles) {
            ks.begin(lds_k[(it + 1) & 1], kb, k.ts, j0 + TK, s.lk - 1, g.D);
            vs.begin(lds_v[(it + 1) & 1], vb, v.ts, j0 + TK, s.lk - 1, g.D);
        }
        if (j0 < wave_hi) {
            const char* tk = lds_k[it & 1];
            const char* tv = lds_v[it & 1];
            f32x16 sc[SUB];
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
                AttnRows<T, DP> kf;
                kf.fetch(tk, (t * KSPLIT + share) * 32 + col, h);
                attn_fence();
                sc[t] = attn_product(kf, qf);
            }
            if (j0 + TK > wave_lo) {
#pragma unroll
                for (int t = 0; t < SUB; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (j0 + (t * KSPLIT + share) * 32 + 8 * (i / 4) + 4 * h + i % 4 >= limit) sc[t][i] = -INFINITY;
                if (g.causal) {
#pragma unroll
                    for (int t = 0; t < SUB; ++t) odd |= attn_odd<T, DP>(tv, (t * KSPLIT + share) * 32, lane);
                }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int t = 0; t < SUB; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[t][i]);
            mx = fmaxf(mx, attn_other_half(mx)) * g.c;
            if (__any(mx > m + 8.f)) {
                const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= f;
#pragma unroll
                for (int db = 0; db < L::DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[db][i] *= f;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int t = 0; t < SUB; ++t) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[t][i] = __builtin_amdgcn_exp2f(fmaf(sc[t][i], g.c, -ref));
                    l += sc[t][i];
                }
                AttnProb<T> p;
                p.set(sc[t]);
#pragma unroll
                for (int db = 0; db < L::DB; ++db) {
                    AttnCols<T, DP> vf;
                    vf.fetch(tv, (t * KSPLIT + share) * 32, db, lane);
                    vf.mma(acc[db], p);
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
    l += attn_other_half(l);
    if (__any(odd))
        attn_redo<T, DP>((const In*)q.p + (size_t)(s.q0 + tok) * q.ts + (size_t)head * q.hs, kb, k.ts, vb, v.ts, acc, g.D, g.c, m, limit, share * 32,
                         KSPLIT * 32, wave_hi, lane);
    if constexpr (KSPLIT == 2) {          // the second wave's sums to the first one, through the tiles nobody needs any more
        float* pass = lds.template join<GROUPS>(wave % GROUPS);
        __shared__ float pass_m[GROUPS][64], pass_l[GROUPS][64];
        if (share) {
#pragma unroll
            for (int db = 0; db < L::DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) pass[(db * 16 + i) * 64 + lane] = acc[db][i];
            pass_m[wave % GROUPS][lane] = m;
            pass_l[wave % GROUPS][lane] = l;
        }
        __syncthreads();
        if (share) return;
        const float m1 = pass_m[wave % GROUPS][lane], mn = fmaxf(m, m1), ref = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
        l = l * f0 + pass_l[wave % GROUPS][lane] * f1;
        m = mn;
#pragma unroll
        for (int db = 0; db < L::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] = acc[db][i] * f0 + pass[(db * 16 + i) * 64 + lane] * f1;
    }
    if (row0 + col >= rows) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    attn_store_row<Out, L::DB>(out + (size_t)(s.q0 + tok) * o_ts + (size_t)head * o_hs, acc, inv, h, g.D);
    if (lse && h == 0) lse[(size_t)(s.q0 + tok) * g.Hq + head] = l > 0.f || l != l ? (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f : -INFINITY;
}

template <typename T, int DP, int NW, int TK, int KSPLIT>
bool launch_k(AttnGeom g, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, void* out, long long o_ts, long long o_hs, float* lse, bool vec,
              hipStream_t stream) {
    constexpr int BM = NW / KSPLIT * 32, SHIFT = BM == 256 ? 8 : BM == 128 ? 7 : 6;
    const int slots = attn_slots((long long)g.Nq * g.G, g.B, SHIFT);
    if (!attn_grid((long long)slots * g.Hk, NW * 64)) return false;
    g.sorted = attn_sorts(g, (long long)g.Nq * g.G, BM);
    typedef typename AttnElem<T>::Out Out;
    constexpr bool THREE = AttnElem<T>::THREE;          // always whole vectors
    if (vec) hipLaunchKernelGGL((packed_attn_fwd_kernel<T, DP, NW, TK, KSPLIT, true>), dim3(slots * g.Hk), dim3(NW * 64), 0, stream, g, q, k, v, (Out*)out, o_ts, o_hs, lse, slots);
    else hipLaunchKernelGGL((packed_attn_fwd_kernel<T, DP, NW, TK, KSPLIT, THREE>), dim3(slots * g.Hk), dim3(NW * 64), 0, stream, g, q, k, v, (Out*)out, o_ts, o_hs, lse, slots);
    return true;
}
template <typename T, int DP, int NW, int TK>
bool launch(const AttnGeom& g, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, void* out, long long o_ts, long long o_hs, float* lse,
            bool vec, hipStream_t stream) {
    constexpr int LOW_NW = AttnElem<T>::THREE ? NW : 2, LOW_TK = AttnElem<T>::THREE ? TK : 32;
    if (TK == 64 && attn_few_blocks(g, NW * 32)) return launch_k<T, DP, NW, TK, TK == 64 ? 2 : 1>(g, q, k, v, out, o_ts, o_hs, lse, vec, stream);
    if (!AttnElem<T>::THREE && attn_low_rows(g)) return launch_k<T, DP, LOW_NW, LOW_TK, 1>(g, q, k, v, out, o_ts, o_hs, lse, vec, stream);
    return launch_k<T, DP, NW, TK, 1>(g, q, k, v, out, o_ts, o_hs, lse, vec, stream);
}

}  // namespace

int attn_geom(AttnGeom& g, const int* off_q, const int* off_k, const int* k_len, float temperature, int causal, int B, int Nq, int Nk, int Hq,
              int Hk, int D, int act) {
    if (B <= 0 || Nq < 0 || Nk < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || D <= 0 || D > 128) return UNCR_ESHAPE;
    if ((long long)Nq * (Hq / Hk) > 0x40000000ll || Nk > 0x40000000) return UNCR_ESHAPE;      // rows and keys are counted in 32 bits
    // beyond these the scale of the scores or its product with a hidden score, -infinity, is no number
    if ((act != 0 && act != 1) || !off_q || !off_k || !(temperature >= 1e-30f && temperature <= 1e30f)) return UNCR_EINVAL;
    // blocks of a launch: at least 32 rows each
    if (((((long long)Nq * (Hq / Hk)) >> 5) + B) * Hk > 0x7fffffffll || (((long long)Nk >> 5) + B) * Hk > 0x7fffffffll) return UNCR_ESHAPE;
    g.off_q = off_q; g.off_k = off_k; g.k_len = k_len;
    g.B = B; g.Nq = Nq; g.Nk = Nk; g.Hq = Hq; g.Hk = Hk; g.G = Hq / Hk; g.D = D;
    g.causal = causal ? 1 : 0;
    g.fill = 0;
    g.scale = 1.f / temperature;
    g.c = (float)(1.4426950408889634 / (double)temperature);
    return UNCR_OK;
}

bool attn_aligned(const AttnTensor* t, int n, int D, int act) {
    const int size = act ? 2 : 4;
    bool ok = (D * size) % 16 == 0;
    for (int i = 0; i < n; ++i) ok = ok && (uintptr_t)t[i].p % 16 == 0 && (t[i].ts * size) % 16 == 0 && (t[i].hs * size) % 16 == 0;
    return ok;
}

extern "C" int uncr_packed_attn_work(int max_q, int max_k, int B, int Nq, int Nk, int Hq, int Hk, int D, int act) {
    AttnGeom g;
    static const int none = 0;
    if (attn_geom(g, &none, &none, nullptr, 1.f, 0, B, Nq, Nk, Hq, Hk, D, act) != UNCR_OK) return 0;
    const AttnSplit s = attn_split(g, max_q, max_k, act);
    if (s.waves) return s.splits > 1 ? (int)((long long)s.splits * Nq * Hq * (D + 2)) : 0;
    return attn_three(g, act, true) ? (int)attn_planes_floats(g, 1, 2) : 0;
}

extern "C" int uncr_packed_attn_fwd(const void* q, long long q_ts, long long q_hs, const void* k, long long k_ts, long long k_hs, const void* v,
                                    long long v_ts, long long v_hs, void* out, long long o_ts, long long o_hs, float* lse, const int* off_q,
                                    const int* off_k, const int* k_len, float temperature, int causal, int fill, int max_q, int max_k,
                                    float* work, long long work_floats, int B, int Nq, int Nk, int Hq, int Hk, int D, int act,
                                    hipStream_t stream) {
    AttnGeom g;
    const int rc = attn_geom(g, off_q, off_k, k_len, temperature, causal, B, Nq, Nk, Hq, Hk, D, act);
    if (rc != UNCR_OK) return rc;
    if (Nq == 0) return UNCR_OK;
    if (!q || !out || (Nk && (!k || !v))) return UNCR_EINVAL;
    g.fill = fill ? 1 : 0;
    const AttnTensor tq = {q, q_ts, q_hs}, tk = {k, k_ts, k_hs}, tv = {v, v_ts, v_hs};
    const AttnTensor all[] = {tq, tk, tv};
    const bool vec = attn_aligned(all, 3, D, act);
    if ((D & 3) == 0) {         // the epilogue's 4-element stores
        const int size = (act ? 2 : 4) * 4;
        if ((uintptr_t)out % size || (o_ts * size / 4) % size || (o_hs * size / 4) % size) return UNCR_EINVAL;
    }
    const AttnSplit split = attn_split(g, max_q, max_k, act);
    bool fits;
    if (split.waves) {
        if (split.splits > 1 && (!work || work_floats < (long long)split.splits * Nq * Hq * (D + 2))) return UNCR_EINVAL;
        fits = attn_rows_fwd(g, split, tq, tk, tv, out, o_ts, o_hs, lse, work, act, vec, stream);
    } else if (attn_three(g, act, vec)) {
        if (!work || work_floats < attn_planes_floats(g, 1, 2)) return UNCR_EINVAL;
        const int n[3] = {Nq, Nk, Nk}, h[3] = {Hq, Hk, Hk};
        AttnTensor p[3];
        attn_planes(g, all, n, h, 3, work, p, stream);
        if (D <= 32) fits = launch<AttnThree, 32, 4, 64>(g, p[0], p[1], p[2], out, o_ts, o_hs, lse, true, stream);
        else fits = launch<AttnThree, 64, 4, 32>(g, p[0], p[1], p[2], out, o_ts, o_hs, lse, true, stream);
    } else if (act) {
        if (D <= 32) fits = launch<__bf16, 32, 4, 64>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
        else if (D <= 64) fits = launch<__bf16, 64, 4, 64>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
        else fits = launch<__bf16, 128, 8, 64>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
    } else {
        if (D <= 32) fits = launch<float, 32, 4, 64>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
        else if (D <= 64) fits = launch<float, 64, 4, 64>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
        else fits = launch<float, 128, 4, 32>(g, tq, tk, tv, out, o_ts, o_hs, lse, vec, stream);
    }
    if (!fits) return UNCR_ESHAPE;
    UNCR_LAUNCH_CHECK();
    return UNCR_OK;
}
