// Attention, forward, gfx950:  o_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j) over the visible keys.
//
// One pass over the keys with the running maximum and sum per row.  A wave owns 32 query rows, a block NW of them; key and
// value tiles of KT rows go through LDS (double-buffered, the next tile's global loads in flight during the current one's
// products), the scores never leave the registers: S^T = K Q^T has the queries as columns, so a lane owns one softmax
// row, and its probabilities are the B fragments of O^T += V^T P^T as they stand (ctn_attn.h).
// Probabilities and output accumulate in fp32; for bf16 tensors the probabilities are rounded to bf16 for the second
// product (relative 2^-8 each at most, averaged over the keys; their sum is taken before the rounding).
// Few rows against many keys: the query heads of a key head become rows of one tile and the key range is split over blocks,
// each leaving its normalised output and its log-sum to the caller's workspace; a second launch joins them.
#include "ctn_attn.h"

namespace {
using namespace attn;

struct fwd_params {
    ctn_attn_args a;
    int G, rows, nqt, heads, nsplit;      // heads: grid heads (H, or Hk when the group is packed into rows)
    bool packed;
    float sl2;                            // scale log2(e)
    float* po; float* pl;                 // split: partial outputs [nsplit][B H Tq][D] and log2-sums [nsplit][B H Tq]
};

template <typename T, int DT, int NW, int KT>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn_fwd_kernel(const fwd_params f) {
    constexpr int NP = Planes<T>::N, NT = NW * 64, KS = DT / 16, NK = KT / 32, ND = DT / 32;
    typedef Tile<T, DT, KT, NT> tile_t;
    constexpr int BUF = 2 * tile_t::BYTES;                       // a buffer: K planes, V planes
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * BUF];
    const ctn_attn_args& a = f.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int off = a.Tk - a.Tq;
    unsigned tile, unit;
    deal(blockIdx.x, a.batch * f.heads, f.nqt * f.nsplit, a.causal, tile, unit);
    const int sp = tile % f.nsplit;
    const int qt = f.nqt - 1 - (int)(tile / f.nsplit);           // with a causal mask the last queries see the most keys
    const int hh = unit % f.heads, b = unit / f.heads;

    const int w0 = (qt * NW + wave) * 32;                        // the wave's first row
    const int n = w0 + (lane & 31);
    const bool live = n < f.rows;
    const int g = f.packed ? n / a.Tq : 0, tq = f.packed ? n - g * a.Tq : n;
    const int hk = f.packed ? hh : hh / f.G, head = f.packed ? hh * f.G + g : hh;
    int len = a.Tk;
    if (a.lengths) len = min(max(a.lengths[b], 0), a.Tk);
    const int vis = !live ? 0 : a.causal ? min(len, tq + off + 1) : len;         // keys 0 .. vis - 1 are visible
    // block: keys below kend are read; wave: tiles below wfull need no mask, tiles from wend on hold nothing for it
    int kend = len, wfull = len, wend = len;
    if (a.causal) {
        const int last = f.packed ? a.Tq - 1 : min(f.rows, (qt + 1) * 32 * NW) - 1;
        kend = min(len, last + off + 1);
        wfull = min(len, (f.packed ? 0 : w0) + off + 1);
        wend = min(len, (f.packed ? a.Tq : min(f.rows, w0 + 32)) + off);
    }
    if (w0 >= f.rows) wend = 0;
    const int ntile = kend > 0 ? (kend + KT - 1) / KT : 0;
    const int t0 = (int)((int64_t)ntile * sp / f.nsplit), t1 = (int)((int64_t)ntile * (sp + 1) / f.nsplit);

    const T* kp = (const T*)a.k + b * a.k_b + hk * a.k_h + (int64_t)t0 * KT * a.k_t;
    const T* vp = (const T*)a.v + b * a.v_b + hk * a.v_h + (int64_t)t0 * KT * a.v_t;
    const int64_t kstep = KT * a.k_t, vstep = KT * a.v_t;
    int left = kend - t0 * KT;
    tile_t tk, tv;
    tk.init(a.k_t, a.D);
    tv.init(a.v_t, a.D);
    auto fetch = [&]() {                                         // the next tile
        tk.load(kp, left, a.D);
        tv.load(vp, left, a.D);
        kp += kstep, vp += vstep, left -= KT;
    };
    auto stage = [&](const int buf) {
        tk.store(lds + buf * BUF);
        tv.store(lds + buf * BUF + tile_t::BYTES);
    };
    if (t0 < t1) fetch();

    Frag<NP> q[KS];
    {
        const T* qp = (const T*)a.q + b * a.q_b + tq * a.q_t + head * a.q_h;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            Chunk<T> c;
            const int d = 16 * s + 8 * half;
            if (live && d < a.D) c.load(qp + d);
            else c.zero();
            c.frag(q[s]);
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    if (t0 < t1) stage(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const unsigned char* K = lds + ((t - t0) & 1) * BUF;
        const unsigned char* V = K + tile_t::BYTES;
        if (t + 1 < t1) fetch();
        if (t * KT < wend) {
            f32x16 s[NK];
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[j][e] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    Frag<NP> k;
                    frag_rows<NP, DT, KT>(K, 32 * j, i, k);
                    mma(s[j], k, q[i]);
                }
            if ((t + 1) * KT > wfull) {
                const int lim = vis - t * KT - 4 * half;
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[j][e] = 32 * j + (e & 3) + 8 * (e >> 2) < lim ? s[j][e] : -INFINITY;
            }
            float mx = s[0][0];
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[j][e]);
            const float mn = fmaxf(m, half_max(mx));
            const float base = mn == -INFINITY ? 0.f : mn * f.sl2;           // rows that see nothing yet stay at zero
            if (__any(mn != m)) {
                const float alpha = __builtin_amdgcn_exp2f(m * f.sl2 - base);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
            }
            m = mn;
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][8 * (i & 1) + e], f.sl2, -base));
                    l += x[e];
                }
                Frag<NP> p;
                make_frag(x, p);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<NP> v;
                    frag_cols<NP, DT, KT>(V, 16 * i, 32 * d, v);
                    mma(o[d], v, p);
                }
            }
        }
        if (t + 1 < t1) stage((t - t0 + 1) & 1);
        __syncthreads();
    }

    l = half_sum(l);
    if (!live) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const float lse = l > 0.f ? m * f.sl2 + __builtin_amdgcn_logf(l) : -INFINITY;
    const int64_t row = ((int64_t)b * a.H + head) * a.Tq + tq, nrow = (int64_t)a.batch * a.H * a.Tq;
    float* po = f.po + (sp * nrow + row) * a.D;
    T* op = (T*)a.o + b * a.o_b + tq * a.o_t + head * a.o_h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int c = 32 * d + acc_row(e);
            const f32x4 v = f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]} * inv;
            if (c < a.D) {
                if (f.nsplit > 1) ctn_st4(po + c, v);
                else store4(op + c, v);
            }
        }
    if (half == 0) {
        if (f.nsplit > 1) f.pl[sp * nrow + row] = lse;
        else if (a.lse) a.lse[row] = lse;
    }
}

// Joins the key ranges of a row: o = sum_s 2^(l_s - max) o_s / sum_s 2^(l_s - max).  One wave per row, lanes along D.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const fwd_params f) {
    const ctn_attn_args& a = f.a;
    const int lane = threadIdx.x & 63;
    const int64_t nrow = (int64_t)a.batch * a.H * a.Tq, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= nrow) return;
    const int tq = row % a.Tq, head = row / a.Tq % a.H;
    const int64_t b = row / a.Tq / a.H;
    float mx = -INFINITY;
    for (int s = 0; s < f.nsplit; ++s) mx = fmaxf(mx, f.pl[s * nrow + row]);
    float tot = 0.f, x[2] = {0.f, 0.f};
    if (mx != -INFINITY)
        for (int s = 0; s < f.nsplit; ++s) {
            const float ls = f.pl[s * nrow + row];
            if (ls == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(ls - mx);
            tot += w;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lane + 64 * i < a.D) x[i] += w * f.po[(s * nrow + row) * a.D + lane + 64 * i];
        }
    const float inv = tot > 0.f ? 1.f / tot : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < a.D) ((T*)a.o + b * a.o_b + tq * a.o_t + head * a.o_h)[lane + 64 * i] = (T)(x[i] * inv);
    if (a.lse && lane == 0) a.lse[row] = tot > 0.f ? mx + __builtin_amdgcn_logf(tot) : -INFINITY;
}

// Keys per tile: 64, halved where the LDS of three planes would keep a third block off the CU (fp32 heads of 64 features,
// 16 x 8 heads of 1000 steps: 183 us against 222 us; of 32: 510 us against 535 us the other way) or the blocks are small.
template <typename T, int DT, int NW> constexpr int key_tile() {
    return Planes<T>::N * DT > 128 || (Planes<T>::N == 3 && NW < 4) ? 32 : 64;
}

// How the call is cut.  Packed: all query heads of a key head in one tile of at most 128 rows, where there are fewer than
// 32 queries (a tile per head would leave most of its 32 rows empty and read the keys once per query head).
struct fwd_cut { bool packed; int rows, nw, nqt, heads, nsplit; };
fwd_cut cut_forward(const ctn_attn_args& a) {
    fwd_cut c;
    const int G = a.H / a.Hk;
    c.packed = G > 1 && a.Tq < 32 && (int64_t)G * a.Tq <= 128;
    c.rows = c.packed ? G * a.Tq : a.Tq;
    c.heads = c.packed ? a.Hk : a.H;
    c.nw = c.rows <= 32 ? 1 : c.rows <= 64 ? 2 : 4;
    c.nqt = ctn_cdiv(c.rows, 32 * c.nw);
    c.nsplit = 1;
    const int64_t blocks = (int64_t)a.batch * c.heads * c.nqt;
    const int tiles = ctn_cdiv(a.Tk, 64);
    if (c.nqt == 1 && blocks < 512) {
        // split the keys until there are about eight waves for every CU, at least four tiles a piece
        int64_t n = 2048 / (blocks * c.nw);
        if (n > tiles / 4) n = tiles / 4;
        if (n > 1) c.nsplit = (int)n;
    }
    return c;
}

template <typename T, int DT, int NW>
void launch_fwd(const fwd_params& f, unsigned grid, hipStream_t s) {
    hipLaunchKernelGGL((attn_fwd_kernel<T, DT, NW, key_tile<T, DT, NW>()>), dim3(grid), dim3(NW * 64), 0, s, f);
}
template <typename T, int DT>
void launch_fwd_nw(const fwd_params& f, int nw, unsigned grid, hipStream_t s) {
    if (nw == 1) launch_fwd<T, DT, 1>(f, grid, s);
    else if (nw == 2) launch_fwd<T, DT, 2>(f, grid, s);
    else launch_fwd<T, DT, 4>(f, grid, s);
}
template <typename T>
void launch_fwd_type(const fwd_params& f, int nw, unsigned grid, hipStream_t s) {
    if (f.a.D <= 32) launch_fwd_nw<T, 32>(f, nw, grid, s);
    else if (f.a.D <= 64) launch_fwd_nw<T, 64>(f, nw, grid, s);
    else launch_fwd_nw<T, 128>(f, nw, grid, s);
}

}  // namespace

bool ctn_attn_args_ok(const ctn_attn_args* a, const char* who) {
    if (!a || (a->type != CTN_TYPE_F32 && a->type != CTN_TYPE_BF16) || a->batch < 0 || a->Tq < 0 || a->Tk < 0 || a->H < 1 ||
        a->Hk < 1 || a->H % a->Hk || a->D < 8 || a->D > 128 || a->D % 8 || !(a->scale > 0.f) || !(a->scale < INFINITY)) {
        ctn_set_error("%s: type / sizes (heads a multiple of key heads, 8 to 128 features in multiples of 8, scale > 0)", who);
        return false;
    }
    if (a->Tq > 0x3fffffff || a->Tk > 0x3fffffff) {
        ctn_set_error("%s: sequences of up to 2^30 tokens", who);
        return false;
    }
    const int es = a->type == CTN_TYPE_F32 ? 4 : 2;
    const bool some = a->batch > 0 && a->Tq > 0, keys = a->batch > 0 && a->Tk > 0;
    if ((some && (!a->q || !attn::strides_ok(a->q, a->q_b, a->q_t, a->q_h, es, a->D, a->Tq) || !a->o ||
                  !attn::strides_ok(a->o, a->o_b, a->o_t, a->o_h, es, a->D, a->Tq))) ||
        (keys && (!a->k || !a->v || !attn::strides_ok(a->k, a->k_b, a->k_t, a->k_h, es, a->D, a->Tk) ||
                  !attn::strides_ok(a->v, a->v_b, a->v_t, a->v_h, es, a->D, a->Tk)))) {
        ctn_set_error("%s: q, k, v, o must be 16-byte aligned with strides of whole 16 bytes and rows that do not overlap, less than 16 MiB apart", who);
        return false;
    }
    return true;
}

extern "C" {

int ctn_sizeof_attn_args(void) { return (int)sizeof(ctn_attn_args); }

int64_t ctn_attn_fwd_ws_floats(const ctn_attn_args* a) {
    if (!ctn_attn_args_ok(a, "ctn_attn_fwd_ws_floats")) return -1;
    if (a->batch == 0 || a->Tq == 0) return 0;
    const fwd_cut c = cut_forward(*a);
    return c.nsplit > 1 ? (int64_t)c.nsplit * a->batch * a->H * a->Tq * (a->D + 1) : 0;
}

int ctn_attn_fwd(const ctn_attn_args* a, void* stream) {
    if (!ctn_attn_args_ok(a, "ctn_attn_fwd")) return CTN_ERR_ARG;
    if (a->batch == 0 || a->Tq == 0) return CTN_OK;
    const fwd_cut c = cut_forward(*a);
    fwd_params f;
    f.a = *a;
    f.G = a->H / a->Hk, f.rows = c.rows, f.nqt = c.nqt, f.heads = c.heads, f.nsplit = c.nsplit, f.packed = c.packed;
    f.sl2 = a->scale * attn::LOG2E;
    const int64_t nrow = (int64_t)a->batch * a->H * a->Tq;
    f.po = f.pl = nullptr;
    if (c.nsplit > 1) {
        CTN_REQUIRE(a->ws && ctn_aligned16(a->ws) && a->ws_floats >= c.nsplit * nrow * (a->D + 1),
                    "ctn_attn_fwd: workspace of %lld floats, %lld needed", (long long)a->ws_floats,
                    (long long)(c.nsplit * nrow * (a->D + 1)));
        f.po = a->ws, f.pl = a->ws + c.nsplit * nrow * a->D;
    }
    const int64_t grid = (int64_t)a->batch * c.heads * c.nqt * c.nsplit;
    CTN_REQUIRE(grid < 0x7fffffff && (nrow + 3) / 4 < 0x7fffffff, "ctn_attn_fwd: too much work for one launch");
    hipStream_t s = (hipStream_t)stream;
    if (a->type == CTN_TYPE_F32) launch_fwd_type<float>(f, c.nw, (unsigned)grid, s);
    else launch_fwd_type<__bf16>(f, c.nw, (unsigned)grid, s);
    CTN_CHECK_LAUNCH("ctn_attn_fwd");
    if (c.nsplit > 1) {
        const dim3 jg((unsigned)((nrow + 3) / 4));
        if (a->type == CTN_TYPE_F32) hipLaunchKernelGGL(attn_join_kernel<float>, jg, dim3(256), 0, s, f);
        else hipLaunchKernelGGL(attn_join_kernel<__bf16>, jg, dim3(256), 0, s, f);
        CTN_CHECK_LAUNCH("ctn_attn_fwd (join)");
    }
    return CTN_OK;
}

}  // extern "C"
