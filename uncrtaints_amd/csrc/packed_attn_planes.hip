// fp32 rows taken apart for the bf16 matrix units (AttnThree in packed_attn.h): [N][H][D] -> [N][H][3][D rounded up to 8] of bf16, zeros
// behind D.  Bound: memory, 4 bytes read and 6 written per element; one launch for all tensors of a call.
#include "packed_attn.h"

namespace {

struct Planes { AttnTensor in[ATTN_MAX_PLANES]; __bf16* out[ATTN_MAX_PLANES]; int N[ATTN_MAX_PLANES], H[ATTN_MAX_PLANES]; };

__global__ __launch_bounds__(256) void attn_planes_kernel(const Planes a, int D) {
    const int z = blockIdx.y, per = (D + 7) / 8, H = a.H[z];
    const long long total = (long long)a.N[z] * H * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / per;
        const int c = (int)(i - row * per);
        const long long t = row / H;
        const float* src = (const float*)a.in[z].p + t * a.in[z].ts + (row - t * H) * a.in[z].hs + c * 8;
        float x[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const f32x4 f = c * 8 + q * 4 < D ? *reinterpret_cast<const f32x4*>(src + q * 4) : (f32x4)(0.f);      // D is a multiple of 4
#pragma unroll
            for (int e = 0; e < 4; ++e) x[q * 4 + e] = f[e];
        }
        bf16x8 v[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // nothing is left of an infinity or NaN, and a number that would round to an infinity keeps its upper bits instead
            __bf16 r = (__bf16)x[e];
            const bool finite = fabsf(x[e]) <= 3.4028234664e38f;
            if (finite && fabsf((float)r) > 3.4028234664e38f) r = (__bf16)__uint_as_float(__float_as_uint(x[e]) & 0xffff0000u);
            float left = finite ? x[e] - (float)r : 0.f;
            v[0][e] = r;
            v[1][e] = (__bf16)left;
            left -= (float)v[1][e];
            v[2][e] = (__bf16)left;
        }
        __bf16* dst = a.out[z] + row * 3 * per * 8 + c * 8;
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(dst + (long long)k * per * 8) = v[k];
    }
}

}  // namespace

// Long fp32 sequences.  The launch before the products costs 10 bytes per element of all tensors, used or not; what it buys grows with the rows
// that meet a key.  Forward, three parts beside fp32 products: 32 sequences of 600 keys, 16/4 heads of 64: 128 rows of each 95 against 125 us, 512 rows
// 230 against 283; 8 of 8192 keys: 512 rows 748 against 1177.  The rule looks at the keys alone, and a few rows over a cache lose by it: 40 rows of
// each, 8 heads of 64, over 8 caches of 8192 keys 628 against 372 us, over 512 used rows of such caches 162 against 30.
bool attn_three(const AttnGeom& g, int act, bool vec) {
    return act == 0 && vec && g.D <= 64 && g.D % 4 == 0 && g.Nq > 0 && g.Nk / g.B >= 512 && attn_planes_floats(g, 2, 2) < (1ll << 30);
}

long long attn_planes_floats(const AttnGeom& g, long long q_like, long long k_like) {
    const long long row = 3ll * ((g.D + 7) / 8 * 8) / 2;
    return q_like * g.Nq * g.Hq * row + k_like * g.Nk * g.Hk * row;
}

void attn_planes(const AttnGeom& g, const AttnTensor* in, const int* N, const int* H, int n, float* work, AttnTensor* out, hipStream_t stream) {
    Planes a = {};
    const int dp = (g.D + 7) / 8 * 8;
    __bf16* at = (__bf16*)work;
    long long most = 0;
    for (int z = 0; z < n; ++z) {
        a.in[z] = in[z];
        a.out[z] = at;
        a.N[z] = N[z];
        a.H[z] = H[z];
        out[z] = {at, 3ll * dp * H[z], 3ll * dp};
        const long long rows = (long long)N[z] * H[z];
        at += rows * 3 * dp;
        most = rows * (dp / 8) > most ? rows * (dp / 8) : most;
    }
    const long long blocks = (most + 255) / 256;
    hipLaunchKernelGGL(attn_planes_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096), n), dim3(256), 0, stream, a, g.D);
}
