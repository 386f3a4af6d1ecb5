// Rotation of head vectors by positions with several axes (date, row, column), alone or behind a norm of queries and keys per head.
//
//   angle(p) = pos[token][axis(p)] * freq(p);   (a, b) -> (a cos - b sin, a sin + b cos)   for the pair p = (a, b) of a head vector
//   norm:  y = R(angle) (w * x * r),  r = 1 / sqrt(mean(x^2) + eps)    (mean over the head's D values)
//   its gradient, u = R(-angle) dy, xhat = x r:   dx = r * (w u - xhat * mean(w u xhat)),   dw = sum over tokens and heads of u * xhat
//
// Bound: memory.  The rotation reads and writes every element once (its gradient is the same kernel with the opposite angle); the norm's
// gradient reads x and dy and recomputes r, so the forward keeps nothing for it.
// Split: a wave takes `tok` tokens and waits for no other.  Their (cos, sin) of every pair are computed ONCE, for all heads of queries and
// keys, into LDS -- the angle in turns in 64 bits (fp32 loses the angle of a far position: 2^-24 * pos * freq radians), reduced, then sincospi
// in fp32.  A group of `lpr` lanes then takes one token and every `strands`-th head: its pairs' (cos, sin) sit in registers, each head is C
// pairs per lane loaded as up to 16-byte vectors.  At least four heads per group where there are that many, so the angles' cost is spread.
// Measured, bf16: 65537 tokens, 40 heads of 128, rotation 262 us (5.1 TB/s; a large copy 4.96); 40001 tokens, 32 + 8 heads of 128, norms and
// rotation 159 us, gradient 245 us and 5 us for the sums of dw (5.1 and 5.0 TB/s).  One token: 3 us.
#include "common.h"

namespace {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_D = 256;
constexpr int ROT_MAX_SLOTS = 1024;     // blocks of the norm's gradient = rows of its dw partials

struct RotGeom {
    const void* pos;         // [N][n_axes]
    const double* turns;     // [D / 2] turns per unit of position of every pair (0: the pair passes through)
    int pos_dt, n_axes;
    int sec0, sec1, sec2, sec3;      // elements per axis; the rest of D passes through
    int neighbours;          // pairs (2i, 2i+1) of the head vector instead of (i, i + n/2) of the axis' section: NB in the kernels
    float sgn;               // +1: rotate, -1: rotate back
    int N, D;
    int chunks;              // D / 2 / C: lanes' work items of one head
    int lpr;                 // lanes per head row (power of two)
    int strands, tok;        // groups of a wave that share a token's heads; tokens per wave
};

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Elem<__bf16> {
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }      // round to nearest even: the one rounding of a store
};

template <typename T, int C> struct alignas(C * sizeof(T) < 16 ? C * sizeof(T) : 16) Pack { T v[C]; };

template <typename T, int C> __device__ __forceinline__ void load(const T* p, float* out) {
    const Pack<T, C> k = *reinterpret_cast<const Pack<T, C>*>(p);
#pragma unroll
    for (int i = 0; i < C; ++i) out[i] = Elem<T>::up(k.v[i]);
}
template <typename T, int C> __device__ __forceinline__ void store(T* p, const float* in) {
    Pack<T, C> k;
#pragma unroll
    for (int i = 0; i < C; ++i) k.v[i] = Elem<T>::down(in[i]);
    *reinterpret_cast<Pack<T, C>*>(p) = k;
}

// The C pairs of work item `j`: elements o1 + i and o2 + i (halves), or o1 + 2i, o1 + 2i + 1 (neighbours)
template <int C, bool NB> __device__ __forceinline__ void place(const RotGeom& g, int j, int& o1, int& o2) {
    int p = j * C;
    if (NB) { o1 = 2 * p; o2 = 0; return; }
    int start = 0, h = g.sec0 >> 1;
    if (p >= h) { p -= h; start += 2 * h; h = g.sec1 >> 1;
        if (p >= h) { p -= h; start += 2 * h; h = g.sec2 >> 1;
            if (p >= h) { p -= h; start += 2 * h; h = g.sec3 >> 1;
                if (p >= h) { p -= h; start += 2 * h; h = (g.D - start) >> 1; } } } }
    o1 = start + p;
    o2 = o1 + h;
}

template <typename T, int C, bool NB> __device__ __forceinline__ void load_pairs(const T* row, int o1, int o2, float* a, float* b) {
    if (NB && C == 1) {
        load<T, 1>(row + o1, a);
        load<T, 1>(row + o1 + 1, b);
    } else if (NB) {
        float x[2 * C];
        load<T, 2 * C>(row + o1, x);
#pragma unroll
        for (int i = 0; i < C; ++i) { a[i] = x[2 * i]; b[i] = x[2 * i + 1]; }
    } else {
        load<T, C>(row + o1, a);
        load<T, C>(row + o2, b);
    }
}
template <typename T, int C, bool NB> __device__ __forceinline__ void store_pairs(T* row, int o1, int o2, const float* a, const float* b) {
    if (NB && C == 1) {
        store<T, 1>(row + o1, a);
        store<T, 1>(row + o1 + 1, b);
    } else if (NB) {
        float x[2 * C];
#pragma unroll
        for (int i = 0; i < C; ++i) { x[2 * i] = a[i]; x[2 * i + 1] = b[i]; }
        store<T, 2 * C>(row + o1, x);
    } else {
        store<T, C>(row + o1, a);
        store<T, C>(row + o2, b);
    }
}

__device__ __forceinline__ double position(const RotGeom& g, int token, int axis) {
    const size_t i = (size_t)token * g.n_axes + axis;
    switch (g.pos_dt) {
        case 0: return (double)((const float*)g.pos)[i];
        case 1: return ((const double*)g.pos)[i];
        case 2: return (double)((const int*)g.pos)[i];
        default: return (double)((const long long*)g.pos)[i];
    }
}

// (cos, sin) of every pair of the wave's tokens into its cs[tok][D / 2]
__device__ __forceinline__ void angles(const RotGeom& g, int token0, float2* cs) {
    const int P = g.D >> 1;
    const int e0 = g.sec0 >> 1, e1 = e0 + (g.sec1 >> 1), e2 = e1 + (g.sec2 >> 1), e3 = e2 + (g.sec3 >> 1);
    for (int i = threadIdx.x & 63; i < g.tok * P; i += 64) {
        const int t = i / P, p = i - t * P;
        float2 v = make_float2(1.f, 0.f);
        if (token0 + t < g.N && p < e3) {
            const int axis = p < e0 ? 0 : p < e1 ? 1 : p < e2 ? 2 : 3;
            const double a = position(g, token0 + t, axis) * g.turns[p];
            float s, c;
            sincospif((float)(2.0 * (a - rint(a))), &s, &c);
            v = make_float2(c, g.sgn * s);
        }
        cs[i] = v;
    }
    __builtin_amdgcn_wave_barrier();      // LDS accesses of a wave are in order: nothing to wait for, only nothing to move across
}

struct HeadSet { const void* x; void* y; const float* w; long long ts, hs, yts, yhs; int H; };

// One pass over queries (and keys): y = R(angle) x, or y = R(angle)(w * x * r).  K work items per lane: two only where C = 1 and D > 128
template <typename T, int C, int K, bool NB, bool NORM>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(const RotGeom g, const HeadSet q, const HeadSet k, float eps) {
    extern __shared__ float2 shared_cs[];
    const int wave = threadIdx.x >> 6;
    float2* cs = shared_cs + wave * g.tok * (g.D >> 1);
    const int token0 = (blockIdx.x * (ROT_THREADS / 64) + wave) * g.tok;
    angles(g, token0, cs);
    const int lane = threadIdx.x & (g.lpr - 1), group = (threadIdx.x & 63) / g.lpr;
    const int t = group / g.strands, strand = group - t * g.strands;
    const int token = token0 + t;
    const bool live = t < g.tok && token < g.N;
    int o1[K], o2[K];
    bool on[K];
    float c[K][C], s[K][C];
#pragma unroll
    for (int m = 0; m < K; ++m) {
        const int j = lane + m * g.lpr;
        on[m] = live && j < g.chunks;
        place<C, NB>(g, on[m] ? j : 0, o1[m], o2[m]);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const float2 v = on[m] ? cs[t * (g.D >> 1) + j * C + i] : make_float2(1.f, 0.f);
            c[m][i] = v.x;
            s[m][i] = v.y;
        }
    }
#pragma unroll
    for (int which = 0; which < (NORM ? 2 : 1); ++which) {
        const HeadSet& z = which ? k : q;
        // heads of queries and keys are dealt to the strands as one list
        int h = strand;
        if (which) { const int past = q.H % g.strands; h = strand >= past ? strand - past : strand - past + g.strands; }
        float wa[K][C], wb[K][C];
        if (NORM) {
#pragma unroll
            for (int m = 0; m < K; ++m) load_pairs<float, C, NB>(z.w, o1[m], o2[m], wa[m], wb[m]);
        }
        for (; h < z.H; h += g.strands) {
            const T* x = (const T*)z.x + (size_t)token * z.ts + (size_t)h * z.hs;
            T* y = (T*)z.y + (size_t)token * z.yts + (size_t)h * z.yhs;
            float a[K][C], b[K][C];
#pragma unroll
            for (int m = 0; m < K; ++m) {
                if (on[m]) load_pairs<T, C, NB>(x, o1[m], o2[m], a[m], b[m]);
                else
#pragma unroll
                    for (int i = 0; i < C; ++i) a[m][i] = b[m][i] = 0.f;
            }
            if (NORM) {
                float ss = 0.f;
#pragma unroll
                for (int m = 0; m < K; ++m)
#pragma unroll
                    for (int i = 0; i < C; ++i) ss = fmaf(a[m][i], a[m][i], fmaf(b[m][i], b[m][i], ss));
                for (int d = g.lpr >> 1; d; d >>= 1) ss += __shfl_xor(ss, d);
                const float r = rsqrtf(ss / (float)g.D + eps);
#pragma unroll
                for (int m = 0; m < K; ++m)
#pragma unroll
                    for (int i = 0; i < C; ++i) { a[m][i] *= r * wa[m][i]; b[m][i] *= r * wb[m][i]; }
            }
#pragma unroll
            for (int m = 0; m < K; ++m) {
                if (!on[m]) continue;
                float u[C], v[C];
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    u[i] = fmaf(a[m][i], c[m][i], -(b[m][i] * s[m][i]));
                    v[i] = fmaf(a[m][i], s[m][i], b[m][i] * c[m][i]);
                }
                store_pairs<T, C, NB>(y, o1[m], o2[m], u, v);
            }
        }
    }
}

struct GradSet { const void* x; const void* dy; void* dx; const float* w; long long ts, hs, gts, ghs; int H; };

// The norm's gradient.  At most four pairs per lane: with eight (164 registers, three waves per SIMD) 40001 tokens x 40 heads x 128 in bf16
// take 320 us, with four (108, four waves) 247 us (5.0 TB/s).  A block walks over token tiles (at most ROT_MAX_SLOTS blocks), dw of queries and keys in registers, and leaves
// one row of partials: their sum in the next launch is in a fixed order, no atomics
template <typename T, int C, int K, bool NB>
__global__ __launch_bounds__(ROT_THREADS) void headnorm_bwd_kernel(const RotGeom g, const GradSet q, const GradSet k, float eps,
                                                                   int tiles, float* __restrict__ part) {
    extern __shared__ float2 shared_cs[];
    __shared__ alignas(16) float red[ROT_THREADS / 64][2][ROT_MAX_D];
    const int wave = threadIdx.x >> 6;
    float2* cs = shared_cs + wave * g.tok * (g.D >> 1);
    const int lane = threadIdx.x & (g.lpr - 1), group = (threadIdx.x & 63) / g.lpr;
    const int t = group / g.strands, strand = group - t * g.strands;
    int o1[K], o2[K];
    float dwa[2][K][C], dwb[2][K][C];
#pragma unroll
    for (int m = 0; m < K; ++m) {
        const int j = lane + m * g.lpr;
        place<C, NB>(g, j < g.chunks ? j : 0, o1[m], o2[m]);
#pragma unroll
        for (int i = 0; i < C; ++i) dwa[0][m][i] = dwb[0][m][i] = dwa[1][m][i] = dwb[1][m][i] = 0.f;
    }
    for (int tile = blockIdx.x * (ROT_THREADS / 64) + wave; tile < tiles; tile += gridDim.x * (ROT_THREADS / 64)) {
        const int token0 = tile * g.tok, token = token0 + t;
        __builtin_amdgcn_wave_barrier();
        angles(g, token0, cs);
        const bool live = t < g.tok && token < g.N;
        bool on[K];
        float c[K][C], s[K][C];
#pragma unroll
        for (int m = 0; m < K; ++m) {
            const int j = lane + m * g.lpr;
            on[m] = live && j < g.chunks;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const float2 v = on[m] ? cs[t * (g.D >> 1) + j * C + i] : make_float2(1.f, 0.f);
                c[m][i] = v.x;
                s[m][i] = v.y;
            }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const GradSet& z = which ? k : q;
            // heads of queries and keys are dealt to the strands as one list
            int h = strand;
            if (which) { const int past = q.H % g.strands; h = strand >= past ? strand - past : strand - past + g.strands; }
            float wa[K][C], wb[K][C];
#pragma unroll
            for (int m = 0; m < K; ++m) load_pairs<float, C, NB>(z.w, o1[m], o2[m], wa[m], wb[m]);
            for (; h < z.H; h += g.strands) {
                const T* x = (const T*)z.x + (size_t)token * z.ts + (size_t)h * z.hs;
                const T* dy = (const T*)z.dy + (size_t)token * z.gts + (size_t)h * z.ghs;
                T* dx = (T*)z.dx + ((size_t)token * z.H + h) * g.D;
                float a[K][C], b[K][C], ua[K][C], ub[K][C];
                float ss = 0.f, dot = 0.f;
#pragma unroll
                for (int m = 0; m < K; ++m) {
                    float ga[C], gb[C];
                    if (on[m]) {
                        load_pairs<T, C, NB>(x, o1[m], o2[m], a[m], b[m]);
                        load_pairs<T, C, NB>(dy, o1[m], o2[m], ga, gb);
                    } else {
#pragma unroll
                        for (int i = 0; i < C; ++i) a[m][i] = b[m][i] = ga[i] = gb[i] = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const float x0 = a[m][i], x1 = b[m][i];
                        const float u0 = fmaf(ga[i], c[m][i], -(gb[i] * s[m][i])), u1 = fmaf(ga[i], s[m][i], gb[i] * c[m][i]);
                        ss = fmaf(x0, x0, fmaf(x1, x1, ss));
                        ua[m][i] = u0 * wa[m][i];
                        ub[m][i] = u1 * wb[m][i];
                        dot = fmaf(ua[m][i], x0, fmaf(ub[m][i], x1, dot));
                        ga[i] = u0 * x0;       // dw terms, still without r
                        gb[i] = u1 * x1;
                    }
                    if (K == 1) {
                        for (int d = g.lpr >> 1; d; d >>= 1) { ss += __shfl_xor(ss, d); dot += __shfl_xor(dot, d); }
                        const float r = rsqrtf(ss / (float)g.D + eps);
#pragma unroll
                        for (int i = 0; i < C; ++i) {
                            if (!on[m]) continue;         // a group behind the last token: r = 1 / sqrt(eps), infinite without eps
                            dwa[which][m][i] = fmaf(ga[i], r, dwa[which][m][i]);
                            dwb[which][m][i] = fmaf(gb[i], r, dwb[which][m][i]);
                        }
                    }
                }
                if (K > 1)
                    for (int d = g.lpr >> 1; d; d >>= 1) { ss += __shfl_xor(ss, d); dot += __shfl_xor(dot, d); }
                const float r = rsqrtf(ss / (float)g.D + eps);
                // mean of w u xhat: with xhat = x r and this every factor stays near the result's size, where x r^3 leaves fp32 for rows of rms
                // 1e13 and more or 1e-13 and less
                const float proj = dot * r / (float)g.D;
#pragma unroll
                for (int m = 0; m < K; ++m) {
                    if (!on[m]) continue;
                    if (K > 1) {
                        float ga[C], gb[C];
                        load_pairs<T, C, NB>(dy, o1[m], o2[m], ga, gb);
#pragma unroll
                        for (int i = 0; i < C; ++i) {
                            const float u0 = fmaf(ga[i], c[m][i], -(gb[i] * s[m][i])), u1 = fmaf(ga[i], s[m][i], gb[i] * c[m][i]);
                            dwa[which][m][i] = fmaf(u0 * a[m][i], r, dwa[which][m][i]);
                            dwb[which][m][i] = fmaf(u1 * b[m][i], r, dwb[which][m][i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        ua[m][i] = r * fmaf(-proj, a[m][i] * r, ua[m][i]);
                        ub[m][i] = r * fmaf(-proj, b[m][i] * r, ub[m][i]);
                    }
                    store_pairs<T, C, NB>(dx, o1[m], o2[m], ua[m], ub[m]);
                }
            }
        }
    }
    // dw of the block: over the groups of a wave by shuffles, over the waves through LDS
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int m = 0; m < K; ++m) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                for (int d = g.lpr; d < 64; d <<= 1) {
                    dwa[which][m][i] += __shfl_xor(dwa[which][m][i], d);
                    dwb[which][m][i] += __shfl_xor(dwb[which][m][i], d);
                }
            const int j = lane + m * g.lpr;
            if ((threadIdx.x & 63) < g.lpr && j < g.chunks)
                store_pairs<float, C, NB>(&red[wave][which][0], o1[m], o2[m], dwa[which][m], dwb[which][m]);
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * g.D; i += ROT_THREADS) {
        const int which = i / g.D, e = i - which * g.D;
        float v = 0.f;
        for (int w = 0; w < ROT_THREADS / 64; ++w) v += red[w][which][e];
        part[(size_t)blockIdx.x * 2 * g.D + i] = v;
    }
}

// dw[i] = sum over the partials' rows, in 64 bits and a fixed order: 16 columns x 64 row strands per block
__global__ __launch_bounds__(1024) void headnorm_dw_kernel(const float* __restrict__ part, int rows, int n, float* __restrict__ dwq,
                                                           float* __restrict__ dwk) {
    __shared__ double acc[64][17];
    const int x = threadIdx.x & 15, c = blockIdx.x * 16 + x, s = threadIdx.x >> 4;
    double v = 0.0;
    if (c < 2 * n)
#pragma unroll 8
        for (int r = s; r < rows; r += 64) v += (double)part[(size_t)r * 2 * n + c];
    acc[s][x] = v;
    __syncthreads();
    for (int h = 32; h; h >>= 1) {
        if (s < h) acc[s][x] += acc[s + h][x];
        __syncthreads();
    }
    if (s == 0 && c < 2 * n) (c < n ? dwq[c] : dwk[c - n]) = (float)acc[0][x];
}

// Pairs per lane: as many as one 16-byte vector holds of one component (halves) or of whole pairs (neighbours), fewer where an axis' half
// section would be cut or a row does not start aligned for it
int pick_c(const RotGeom& g, const long long* strides, int n_strides, const void* const* ptrs, int n_ptrs, int size, int max_c, const float* wq = nullptr,
           const float* wk = nullptr) {
    const int halves[5] = {g.sec0 / 2, g.sec1 / 2, g.sec2 / 2, g.sec3 / 2, (g.D - g.sec0 - g.sec1 - g.sec2 - g.sec3) / 2};
    const int wide = (g.neighbours ? 8 : 16) / size;
    for (int c = wide < max_c ? wide : max_c; c > 1; c >>= 1) {
        const int align = c * size * (g.neighbours ? 2 : 1);
        bool ok = (g.D / 2) % c == 0;
        if (!g.neighbours)
            for (int h : halves) ok = ok && h % c == 0;
        for (int i = 0; i < n_strides; ++i) ok = ok && (strides[i] * size) % align == 0;
        for (int i = 0; i < n_ptrs; ++i) ok = ok && ((uintptr_t)ptrs[i] % align) == 0;
        ok = ok && (((uintptr_t)wq | (uintptr_t)wk) % (align * 4 / size < 16 ? align * 4 / size : 16)) == 0;
        if (ok) return c;
    }
    return 1;          // one element at a time
}

// lanes per row, groups, tokens per wave for C pairs per lane and `heads` heads
int shape(RotGeom& g, int c, int heads) {
    g.chunks = g.D / 2 / c;
    g.lpr = 1;
    while (g.lpr < g.chunks && g.lpr < 64) g.lpr <<= 1;
    const int groups = 64 / g.lpr;
    g.strands = 1;
    while (g.strands < groups && g.strands * 8 <= heads) g.strands <<= 1;
    g.tok = groups / g.strands;
    return (g.chunks + g.lpr - 1) / g.lpr;
}

int geom(RotGeom& g, const void* pos, int pos_dt, int n_axes, int s0, int s1, int s2, int s3, const double* turns, int neighbours, int inverse,
         int N, int D) {
    if (N < 0 || D <= 0 || D > ROT_MAX_D || (D & 1)) return UNCR_ESHAPE;
    if (n_axes < 0 || n_axes > 4 || pos_dt < 0 || pos_dt > 3) return UNCR_EINVAL;
    const int s[4] = {s0, s1, s2, s3};
    long long sum = 0;
    for (int i = 0; i < 4; ++i) {
        if (s[i] < 0 || (s[i] & 1) || (i >= n_axes && s[i])) return UNCR_ESHAPE;
        sum += s[i];
    }
    if (sum > D) return UNCR_ESHAPE;
    if (sum && N && (!pos || !turns)) return UNCR_EINVAL;
    g.pos = pos; g.turns = turns; g.pos_dt = pos_dt; g.n_axes = n_axes;
    g.sec0 = s0; g.sec1 = s1; g.sec2 = s2; g.sec3 = s3;
    g.neighbours = neighbours ? 1 : 0; g.sgn = inverse ? -1.f : 1.f;
    g.N = N; g.D = D;
    return UNCR_OK;
}

struct Fwd { static constexpr int MAX_C = 8; RotGeom g; HeadSet q, k; float eps; int items; hipStream_t stream; };
struct Bwd { static constexpr int MAX_C = 4; RotGeom g; GradSet q, k; float eps; int items, blocks, tiles; float* part; hipStream_t stream; };

size_t lds_bytes(const RotGeom& g) { return (size_t)(ROT_THREADS / 64) * g.tok * (g.D / 2) * sizeof(float2); }

// tokens of a block; the threads of a forward launch are counted in 32 bits
int per_block(const RotGeom& g) { return g.tok * (ROT_THREADS / 64); }
bool fits(const RotGeom& g) { return ((long long)g.N + per_block(g) - 1) / per_block(g) * ROT_THREADS <= 0xffffffffll; }

template <typename T, bool NB, bool NORM, int C, int K> void run(const Fwd& f) {
    const int per = per_block(f.g);
    hipLaunchKernelGGL((rotary_kernel<T, C, K, NB, NORM>), dim3((unsigned)(((long long)f.g.N + per - 1) / per)), dim3(ROT_THREADS), lds_bytes(f.g), f.stream, f.g, f.q, f.k, f.eps);
}
template <typename T, bool NB, bool NORM, int C, int K> void run(const Bwd& b) {
    hipLaunchKernelGGL((headnorm_bwd_kernel<T, C, K, NB>), dim3(b.blocks), dim3(ROT_THREADS), lds_bytes(b.g), b.stream, b.g, b.q, b.k, b.eps, b.tiles, b.part);
}
// the widest vector is 16 bytes: 16 / size pairs of halves, 8 / size pairs of neighbours
template <typename T, bool NB, bool NORM, typename Job> void launch_c(const Job& j, int c) {
    constexpr int WIDE = (NB ? 8 : 16) / sizeof(T), TOP = WIDE < Job::MAX_C ? WIDE : Job::MAX_C;
    if (c == 8) run<T, NB, NORM, TOP >= 8 ? 8 : 1, 1>(j);
    else if (c == 4) run<T, NB, NORM, TOP >= 4 ? 4 : 1, 1>(j);
    else if (c == 2) run<T, NB, NORM, TOP >= 2 ? 2 : 1, 1>(j);
    else if (j.items > 1) run<T, NB, NORM, 1, 2>(j);
    else run<T, NB, NORM, 1, 1>(j);
}
template <bool NORM, typename Job> void launch(const Job& j, int c, int act) {
    if (act) j.g.neighbours ? launch_c<__bf16, true, NORM>(j, c) : launch_c<__bf16, false, NORM>(j, c);
    else j.g.neighbours ? launch_c<float, true, NORM>(j, c) : launch_c<float, false, NORM>(j, c);
}

}  // namespace

extern "C" int uncr_rotary_axes(const void* x, long long x_ts, long long x_hs, void* y, long long y_ts, long long y_hs, const void* pos,
                                int pos_dt, int n_axes, int sec0, int sec1, int sec2, int sec3, const double* turns, int neighbours,
                                int inverse, int N, int H, int D, int act, hipStream_t stream) {
    RotGeom g;
    const int rc = geom(g, pos, pos_dt, n_axes, sec0, sec1, sec2, sec3, turns, neighbours, inverse, N, D);
    if (rc != UNCR_OK) return rc;
    if (H <= 0) return UNCR_ESHAPE;
    if (act != 0 && act != 1) return UNCR_EINVAL;
    if (N == 0) return UNCR_OK;
    if (!x || !y) return UNCR_EINVAL;
    const long long st[] = {x_ts, x_hs, y_ts, y_hs};
    const void* const pt[] = {x, y};
    const int c = pick_c(g, st, 4, pt, 2, act ? 2 : 4, Fwd::MAX_C), items = shape(g, c, H);
    const HeadSet q = {x, y, nullptr, x_ts, x_hs, y_ts, y_hs, H}, none = {nullptr, nullptr, nullptr, 0, 0, 0, 0, 0};
    if (!fits(g)) return UNCR_ESHAPE;
    launch<false>(Fwd{g, q, none, 0.f, items, stream}, c, act);
    UNCR_LAUNCH_CHECK();
    return UNCR_OK;
}

extern "C" int uncr_headnorm_rotary_fwd(const void* q, long long q_ts, long long q_hs, const void* k, long long k_ts, long long k_hs,
                                        const float* wq, const float* wk, float eps, void* qo, void* ko, const void* pos, int pos_dt,
                                        int n_axes, int sec0, int sec1, int sec2, int sec3, const double* turns, int neighbours, int N,
                                        int Hq, int Hk, int D, int act, hipStream_t stream) {
    RotGeom g;
    const int rc = geom(g, pos, pos_dt, n_axes, sec0, sec1, sec2, sec3, turns, neighbours, 0, N, D);
    if (rc != UNCR_OK) return rc;
    if (Hq <= 0 || Hk <= 0) return UNCR_ESHAPE;
    if ((act != 0 && act != 1) || !(eps >= 0.f)) return UNCR_EINVAL;
    if (N == 0) return UNCR_OK;
    if (!q || !k || !wq || !wk || !qo || !ko) return UNCR_EINVAL;
    const long long st[] = {q_ts, q_hs, k_ts, k_hs, (long long)D};
    const void* const pt[] = {q, k, qo, ko};
    const int c = pick_c(g, st, 5, pt, 4, act ? 2 : 4, Fwd::MAX_C, wq, wk), items = shape(g, c, Hq + Hk);
    const HeadSet zq = {q, qo, wq, q_ts, q_hs, (long long)Hq * D, D, Hq}, zk = {k, ko, wk, k_ts, k_hs, (long long)Hk * D, D, Hk};
    if (!fits(g)) return UNCR_ESHAPE;
    launch<true>(Fwd{g, zq, zk, eps, items, stream}, c, act);
    UNCR_LAUNCH_CHECK();
    return UNCR_OK;
}

extern "C" int uncr_headnorm_slots(int N) { return N < ROT_MAX_SLOTS ? (N > 0 ? N : 1) : ROT_MAX_SLOTS; }

extern "C" int uncr_headnorm_rotary_bwd(const void* q, long long q_ts, long long q_hs, const void* k, long long k_ts, long long k_hs,
                                        const float* wq, const float* wk, float eps, const void* gq, long long gq_ts, long long gq_hs,
                                        const void* gk, long long gk_ts, long long gk_hs, void* dq, void* dk, float* part, float* dwq,
                                        float* dwk, const void* pos, int pos_dt, int n_axes, int sec0, int sec1, int sec2, int sec3,
                                        const double* turns, int neighbours, int N, int Hq, int Hk, int D, int act, hipStream_t stream) {
    RotGeom g;
    const int rc = geom(g, pos, pos_dt, n_axes, sec0, sec1, sec2, sec3, turns, neighbours, 1, N, D);
    if (rc != UNCR_OK) return rc;
    if (Hq <= 0 || Hk <= 0) return UNCR_ESHAPE;
    if ((act != 0 && act != 1) || !(eps >= 0.f) || !dwq || !dwk || !part) return UNCR_EINVAL;
    int blocks = 0;
    if (N > 0) {
        if (!q || !k || !wq || !wk || !gq || !gk || !dq || !dk) return UNCR_EINVAL;
        const long long st[] = {q_ts, q_hs, k_ts, k_hs, gq_ts, gq_hs, gk_ts, gk_hs, (long long)D};
        const void* const pt[] = {q, k, gq, gk, dq, dk};
        const int c = pick_c(g, st, 9, pt, 6, act ? 2 : 4, Bwd::MAX_C, wq, wk), items = shape(g, c, Hq + Hk);
        // a wave's tiles; their numbers are counted in 32 bits, up to a round of all waves behind the last one
        const long long tiles = ((long long)N + g.tok - 1) / g.tok, wanted = ((long long)N + per_block(g) - 1) / per_block(g);
        blocks = wanted < ROT_MAX_SLOTS ? (int)wanted : ROT_MAX_SLOTS;
        if (tiles + (long long)blocks * (ROT_THREADS / 64) > 0x7fffffffll) return UNCR_ESHAPE;
        const GradSet zq = {q, gq, dq, wq, q_ts, q_hs, gq_ts, gq_hs, Hq}, zk = {k, gk, dk, wk, k_ts, k_hs, gk_ts, gk_hs, Hk};
        launch<true>(Bwd{g, zq, zk, eps, items, blocks, (int)tiles, part, stream}, c, act);
        UNCR_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(headnorm_dw_kernel, dim3((2 * D + 15) / 16), dim3(1024), 0, stream, part, blocks, D, dwq, dwk);
    UNCR_LAUNCH_CHECK();
    return UNCR_OK;
}
