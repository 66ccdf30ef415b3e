// Rotary positions, gfx950: every pair (a, b) of a head's leading `rotary` elements is turned by 2 pi position turns[pair],
//   a' = m (a cos - b sin),  b' = m (a sin + b cos)      (inverse: sin -> -sin, which is the gradient's map as well)
// pairs are (i, i + rotary / 2) in the half layout, (2 i, 2 i + 1) interleaved; the remaining elements are copied.
//
// Bound by reading x and writing y once.  A thread owns one 16-byte chunk of a head (half layout: one chunk and its partner
// half a rotation further) at one token, forms the chunk's sines once and walks heads -- and, when the batch shares its
// positions, batch elements -- with them.  The angle is a product in 64 bits of which only the distance to the nearest
// quarter turn (below 1/8) goes on in fp32: positions far along a context lose no digits.  Sine and cosine of that
// remainder are their Taylor sums on [-pi/4, pi/4], cut where the next term is below 2e-9.
#include "ctn_common.h"

namespace {

typedef __bf16 xbf16x8 __attribute__((ext_vector_type(8)));
template <typename T> struct XVec;
template <> struct XVec<float> { static constexpr int V = 4; typedef f32x4 type; };
template <> struct XVec<__bf16> { static constexpr int V = 8; typedef xbf16x8 type; };

template <typename T>
__device__ __forceinline__ typename XVec<T>::type xload(const T* __restrict__ p, const int n) {
    constexpr int V = XVec<T>::V;
    typename XVec<T>::type t;
    if (n >= V) {
        __builtin_memcpy(&t, p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = i < n ? p[i] : (T)0.f;
    }
    return t;
}
template <typename T>
__device__ __forceinline__ void xstore(T* __restrict__ p, const int n, const float (&v)[XVec<T>::V]) {
    constexpr int V = XVec<T>::V;
    if (n >= V) {
        typename XVec<T>::type t;
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = (T)v[i];
        __builtin_memcpy(p, &t, 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// sine and cosine of 2 pi u
__device__ __forceinline__ void turn_sincos(const double u, float& s, float& c) {
    const double q = rint(4.0 * u);
    const float t = (float)(u - 0.25 * q) * 6.283185307179586f;
    const float t2 = t * t;
    const float sn = t * (1.f + t2 * (-1.f / 6 + t2 * (1.f / 120 + t2 * (-1.f / 5040 + t2 * (1.f / 362880)))));
    const float cs = 1.f + t2 * (-0.5f + t2 * (1.f / 24 + t2 * (-1.f / 720 + t2 * (1.f / 40320 + t2 * (-1.f / 3628800)))));
    const int k = (int)(q - 4.0 * floor(0.25 * q));             // quarter turns, 0 .. 3
    const float a = (k & 1) ? cs : sn, b = (k & 1) ? sn : cs;
    s = (k & 2) ? -a : a;
    c = (k == 1 || k == 2) ? -b : b;
}

struct rotary_args {
    const void* x; void* y;
    int64_t xbs, xts, xhs, ybs, yts, yhs;
    const int64_t* positions; int64_t pbs, first;
    const double* turns;
    int B, T, H, D, pairs, nrot, nchunk, hs, bper;   // nrot chunks with pairs, nchunk in all; hs heads side by side
    float magnitude, sign;
};

template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const rotary_args a) {
    constexpr int V = XVec<T>::V, NP = INTERLEAVED ? V / 2 : V;
    const unsigned item = blockIdx.x * 256u + threadIdx.x;
    const int c = (int)(item % (unsigned)a.nchunk);
    const unsigned rest = item / (unsigned)a.nchunk;
    const int h0 = (int)(rest % (unsigned)a.hs);
    const int64_t t = rest / (unsigned)a.hs;
    if (t >= a.T) return;
    const int b0 = blockIdx.y * a.bper, b1 = b0 + a.bper < a.B ? b0 + a.bper : a.B;
    const bool rot = c < a.nrot;
    const int p0 = c * NP, np = a.pairs - p0;                     // first pair of the chunk, pairs from there on
    // first element, and how many of the chunk's V elements exist
    const int e0 = rot ? (INTERLEAVED ? c * V : p0) : 2 * a.pairs + (c - a.nrot) * V;
    const int ne = rot ? (INTERLEAVED ? 2 * np : np) : a.D - e0;
    float sn[NP], cs[NP];
    for (int b = b0; b < b1; ++b) {
        if (rot && (b == b0 || a.pbs != 0)) {
            const int64_t pos = a.positions ? a.positions[b * a.pbs + t] : a.first + t;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                turn_sincos(i < np ? (double)pos * a.turns[p0 + i] : 0.0, sn[i], cs[i]);
                sn[i] *= a.magnitude * a.sign;
                cs[i] *= a.magnitude;
            }
        }
        // four heads at a time: their loads are in flight together
        const T* x = (const T*)a.x + b * a.xbs + t * a.xts + e0;
        T* y = (T*)a.y + b * a.ybs + t * a.yts + e0;
        for (int hb = h0; hb < a.H; hb += 4 * a.hs) {
            typename XVec<T>::type r[4], q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int h = hb + k * a.hs;
                if (h < a.H) {
                    r[k] = xload<T>(x + h * a.xhs, ne);
                    if (!INTERLEAVED && rot) q[k] = xload<T>(x + h * a.xhs + a.pairs, ne);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int h = hb + k * a.hs;
                if (h >= a.H) break;
                T* d = y + h * a.yhs;
                float v[V], o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = (float)r[k][i];
                if (!rot) {
                    xstore<T>(d, ne, v);
                } else if (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < V / 2; ++i) {
                        o[2 * i] = v[2 * i] * cs[i] - v[2 * i + 1] * sn[i];
                        o[2 * i + 1] = v[2 * i] * sn[i] + v[2 * i + 1] * cs[i];
                    }
                    xstore<T>(d, ne, o);
                } else {
                    float o2[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int j = i < NP ? i : 0;
                        const float w = (float)q[k][i];
                        o[i] = v[i] * cs[j] - w * sn[j];
                        o2[i] = v[i] * sn[j] + w * cs[j];
                    }
                    xstore<T>(d, ne, o);
                    xstore<T>(d + a.pairs, ne, o2);
                }
            }
        }
    }
}

}  // namespace

extern "C" int ctn_rotary(const void* x, int64_t xbs, int64_t xts, int64_t xhs, int B, int T, int H, int D, int type,
                          const int64_t* positions, int64_t pbs, int64_t first, const double* turns, int rotary, int interleaved,
                          int inverse, float magnitude, void* y, int64_t ybs, int64_t yts, int64_t yhs, void* stream) {
    CTN_REQUIRE(type == CTN_TYPE_F32 || type == CTN_TYPE_BF16, "ctn_rotary: type %d", type);
    CTN_REQUIRE(B >= 0 && T >= 0 && H >= 0 && D > 0 && rotary >= 0 && rotary <= D && rotary % 2 == 0,
                "ctn_rotary: B %d, T %d, H %d, D %d, %d rotated elements (an even number up to D)", B, T, H, D, rotary);
    if (B == 0 || T == 0 || H == 0) return CTN_OK;
    CTN_REQUIRE(x && y && (turns || rotary == 0), "ctn_rotary: null pointer");
    const int V = type == CTN_TYPE_F32 ? 4 : 8;
    rotary_args a;
    a.x = x, a.y = y, a.xbs = xbs, a.xts = xts, a.xhs = xhs, a.ybs = ybs, a.yts = yts, a.yhs = yhs;
    a.positions = positions, a.pbs = positions ? pbs : 0, a.first = first, a.turns = turns;
    a.B = B, a.T = T, a.H = H, a.D = D, a.pairs = rotary / 2;
    a.nrot = ctn_cdiv(interleaved ? rotary : rotary / 2, V);
    a.nchunk = a.nrot + ctn_cdiv(D - rotary, V);
    a.magnitude = magnitude, a.sign = inverse ? -1.f : 1.f;
    // heads side by side: a wave's worth of one token, the rest of the heads reuse the sines
    a.hs = 64 / a.nchunk < 1 ? 1 : 64 / a.nchunk;
    if (a.hs > H) a.hs = H;
    const int64_t blocks = ((int64_t)T * a.hs * a.nchunk + 255) / 256;
    // batch elements per block: as many as share positions, as long as 8 blocks a CU remain
    a.bper = 1;
    if (a.pbs == 0)
        while (a.bper < 16 && a.bper < B && blocks * (B / (2 * a.bper)) >= 2048) a.bper *= 2;
    while (ctn_cdiv(B, a.bper) > 65535) a.bper *= 2;             // the grid's second dimension ends there
    CTN_REQUIRE(blocks < 0xffffff, "ctn_rotary: too many tokens for one launch");
    const dim3 grid((unsigned)blocks, (unsigned)ctn_cdiv(B, a.bper));
    hipStream_t s = (hipStream_t)stream;
    if (type == CTN_TYPE_F32) {
        if (interleaved) hipLaunchKernelGGL((rotary_kernel<float, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rotary_kernel<float, false>), grid, dim3(256), 0, s, a);
    } else {
        if (interleaved) hipLaunchKernelGGL((rotary_kernel<__bf16, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rotary_kernel<__bf16, false>), grid, dim3(256), 0, s, a);
    }
    CTN_CHECK_LAUNCH("ctn_rotary");
    return CTN_OK;
}
