// RMS norms of every query and key head with the rotation of rotary positions in the same pass, and
// rotary positions with several axes (time, height, width); token-major in, head-major out, and the
// gradients back. Per head row x of D elements, halves a = x[0 .. D/2), b = x[D/2 .. D):
//   norm:      r = 1 / sqrt(mean(x^2) + eps),  y = x r w           (or y = x without norms)
//   rotation:  out_a = y_a cos_a - y_b sin_a,  out_b = y_b cos_b + y_a sin_b
//   back:      n_a = g_a cos_a + g_b sin_b,    n_b = g_b cos_b - g_a sin_a
//              dw = sum over tokens and heads of n x r,  dx = r (n w - x r^2 mean(n w x))
// in fp32, one rounding at the end. cos and sin are tables [tokens, D], or formed here: frequency j
// turns by pos[axis(j)] inv_freq[j], axis(j) by consecutive sections or interleaved. The angle is
// kept in turns as a 64-bit fixed-point fraction: inv_freq / 2 pi (fp64, 53 bits) becomes a fraction
// of 2^64, its product with the integer position wraps where whole turns drop out, and the top 32
// bits go to sincospi. At position 2^20 the product is within 2^-33 radians; an fp32 product of
// position and frequency would be off by 2^-5.
//
// Bound: HBM (read and write of q and k, in the backward gradients, q and k in and dq, dk out): 8192 tokens of
// 28 + 4 heads of 128, bf16, with norms: forward 30 to 32 us with q and k from memory (4.8 to 4.5 TB/s), 25 with them in
// the last cache, backward 39 to 41 (5.4 to 5.1 TB/s) and 4 for the sums of dw; three axes without norms over 4096 tokens,
// fp16, 16.2 and 16.8 us from memory (4.2 and 4.0 TB/s), 12.4 and 12.5 from that cache; a large copy reaches 5.2.
// At 830 tokens 4.5 and 7.2 us, a few memory round trips.
// Layout: a lane holds eight elements of a and their eight partners of b (two 16-byte loads, the
// rotation and most of the norm's sum need no other lane), LPH lanes a head, 64 / LPH heads a pass. A
// wave serves one pass -- so each lane has one head, its weights stay in registers and the
// sums of dw too -- and a stream of tokens, the next token's loads in flight during the arithmetic of
// one. Formed angles are shared through LDS: a lane computes one frequency, all read eight.
// The sums of dw go through LDS (shuffles for them took 2 us of a launch at 830 tokens) and one slab a
// work-group, and are added in work-group order by a second launch: no atomics, the same bits every run.
// Capping the registers for more waves (80 forward, 128 backward) spilled and took 45 and 78 us.
#include "elem.h"

namespace dk {

constexpr int kQkThreads = 256;
constexpr int kQkWaves = kQkThreads / kWave;

// sum over the LPH lanes of a head (all get it)
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = 1; o < LPH; o *= 2) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ float8_t load_weight8(const void* w, int dtype, int at) {
    if (dtype == DK_FP32) return load8<DK_FP32>((const float*)w + at);
    if (dtype == DK_BF16) return load8<DK_BF16>((const __bf16*)w + at);
    return load8<DK_FP16>((const _Float16*)w + at);
}

__device__ __forceinline__ int axis_of(const QkRopeArgs& a, int j) {
    if (a.interleaved) {
        const int x = j % a.n_axes;
        return j < a.n_axes * a.section[x] ? x : 0;
    }
    int x = 0, end = a.section[0];
    while (j >= end && x + 1 < a.n_axes) end += a.section[++x];
    return x;
}

template <int DT, int LPH, bool NORM, bool AXES, bool BWD>
__global__ __launch_bounds__(kQkThreads) void qk_rope_kernel(const QkRopeArgs a) {
    typedef typename Elem<DT>::type elem_t;
    typedef typename Elem<DT>::vec vec_t;
    constexpr int HPW = kWave / LPH;                       // heads a pass
    constexpr int NF = LPH * 8 > kWave ? LPH * 8 / kWave : 1;  // frequencies a lane computes
    __shared__ float2_t trig[AXES ? kQkWaves : 1][AXES ? LPH * 8 : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int w = blockIdx.x * kQkWaves + wave;
    const int pass = w % a.passes, stream = w / a.passes;
    const int half = a.d / 2, c = 8 * (lane % LPH);  // this lane's elements c .. c + 7 and half + c ..
    const int slot = pass * HPW + lane / LPH;
    const bool isq = slot < a.hq;
    const int head = isq ? slot : slot - a.hq, heads = isq ? a.hq : a.hk;
    const bool active = c < half && slot < a.hq + a.hk;
    const elem_t* const x_base = (const elem_t*)(isq ? a.q : a.k) + (int64_t)head * a.d + c;
    const int64_t ldx = isq ? a.ldq : a.ldk;
    const elem_t* const g_base = (const elem_t*)(isq ? a.gq : a.gk) + c;
    elem_t* const o_base = (elem_t*)(isq ? a.oq : a.ok) + c;
    const int64_t ldo = isq ? a.ldoq : a.ldok;

    float8_t wa = {}, wb = {}, da = {}, db = {};
    if (NORM && active) {
        const void* const wp = isq ? a.qw : a.kw;
        wa = load_weight8(wp, a.w_dtype, c);
        wb = load_weight8(wp, a.w_dtype, half + c);
    }
    uint64_t freq[NF];
    int64_t pos_at[NF];
    if constexpr (AXES) {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int j = min(lane + kWave * f, half - 1);
            freq[f] = turn_fraction(a.inv_freq[j]);
            pos_at[f] = (int64_t)axis_of(a, j) * a.pos_axis;
        }
    }

    // a token's loads: x (or the gradient, then x), positions
    vec_t na = {}, nb = {}, xa = {}, xb = {};
    int64_t npos[NF];
    const auto fetch = [&](uint32_t row) {
        const uint32_t b = row / a.tokens, t = row - b * a.tokens;
        if (active) {
            if constexpr (BWD) {
                const elem_t* const g = g_base + ((int64_t)(b * (int64_t)heads + head) * a.tokens + t) * a.d;
                na = load8_raw<DT>(g);
                nb = load8_raw<DT>(g + half);
            }
            if constexpr (!BWD || NORM) {
                const elem_t* const x = x_base + (int64_t)row * ldx;
                xa = load8_raw<DT>(x);
                xb = load8_raw<DT>(x + half);
            }
        }
        if constexpr (AXES) {
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int64_t at = pos_at[f] + (int64_t)b * a.pos_batch + t;
                npos[f] = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
            }
        }
    };

    uint32_t row = stream;
    if (stream < a.streams && row < a.rows) fetch(row);
    for (; stream < a.streams && row < a.rows; row += a.streams) {
        const uint32_t b = row / a.tokens, t = row - b * a.tokens;
        float8_t ca, cb, sa, sb;
        if constexpr (AXES) {
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int32_t turn = (int32_t)((freq[f] * (uint64_t)npos[f]) >> 32);
                float s, co;
                sincospif((float)turn * 4.656612873077393e-10f, &s, &co);  // 2^-31 half turns
                if (lane + kWave * f < LPH * 8) trig[wave][lane + kWave * f] = float2_t{co, s};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2_t cs = trig[wave][c + e];
                ca[e] = cb[e] = cs.x;
                sa[e] = sb[e] = cs.y;
            }
            __builtin_amdgcn_wave_barrier();
        } else {
            const int64_t at = (int64_t)b * a.table_batch + (int64_t)t * a.d + (c < half ? c : 0);
            ca = load8<DK_FP32>(a.cos + at);
            sa = load8<DK_FP32>(a.sin + at);
            cb = load8<DK_FP32>(a.cos + at + half);
            sb = load8<DK_FP32>(a.sin + at + half);
        }
        float8_t va = widen8<DT>(BWD ? na : xa), vb = widen8<DT>(BWD ? nb : xb);
        float8_t fa = {}, fb = {};
        if (BWD && NORM) {
            fa = widen8<DT>(xa);
            fb = widen8<DT>(xb);
        }
        const uint32_t next = row + a.streams;
        if (next < a.rows) fetch(next);

        float8_t oa, ob;
        if constexpr (!BWD) {
            if constexpr (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += va[e] * va[e] + vb[e] * vb[e];
                const float r = rsqrtf(head_sum<LPH>(ss) * a.inv_d + a.eps);
                va = va * r * wa;
                vb = vb * r * wb;
            }
            oa = va * ca - vb * sa;
            ob = vb * cb + va * sb;
            if (active) {
                elem_t* const o = o_base + ((int64_t)(b * (int64_t)heads + head) * a.tokens + t) * a.d;
                store8<DT>(o, oa);
                store8<DT>(o + half, ob);
            }
        } else {
            oa = va * ca + vb * sb;
            ob = vb * cb - va * sa;
            if constexpr (NORM) {
                float ss = 0.0f, m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += fa[e] * fa[e] + fb[e] * fb[e];
                const float r = rsqrtf(head_sum<LPH>(ss) * a.inv_d + a.eps);
                fa = fa * r;  // the normalized row
                fb = fb * r;
                da = da + oa * fa;
                db = db + ob * fb;
                oa = oa * wa;
                ob = ob * wb;
#pragma unroll
                for (int e = 0; e < 8; ++e) m += oa[e] * fa[e] + ob[e] * fb[e];
                m = head_sum<LPH>(m) * a.inv_d;
                oa = (oa - fa * m) * r;
                ob = (ob - fb * m) * r;
            }
            if (active) {
                elem_t* const o = o_base + (int64_t)row * ldo + (int64_t)head * a.d;
                store8<DT>(o, oa);
                store8<DT>(o + half, ob);
            }
        }
    }

    if constexpr (BWD && NORM) {
        if (a.slabs == nullptr) return;
        // this work-group's sums of dw, over the heads of its waves' passes in order
        __shared__ float sums[kQkWaves][kWave][17];  // 17: both sides of the exchange spread over the banks
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sums[wave][lane][e] = active ? da[e] : 0.0f;
            sums[wave][lane][8 + e] = active ? db[e] : 0.0f;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * a.d; i += kQkThreads) {
            const int side = i >= a.d, d = side ? i - a.d : i, c0 = d < half ? d : d - half;
            const int at = c0 / 8, e = (d < half ? 0 : 8) + c0 % 8;
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < kQkWaves; ++k) {
                const int first = (blockIdx.x * kQkWaves + k) % a.passes * HPW;
#pragma unroll
                for (int h = 0; h < HPW; ++h)
                    if ((first + h >= a.hq) == side) v += sums[k][h * LPH + at][e];
            }
            a.slabs[(int64_t)blockIdx.x * 2 * a.d + i] = v;
        }
    }
}

// dw of q (columns 0 .. d - 1 of a slab) and k (d .. 2 d - 1): slabs added by 64 threads a column, each in
// slab order, then those in a fixed order
constexpr int kSlabCols = 16, kSlabRows = 64;
__global__ __launch_bounds__(kSlabCols* kSlabRows) void norm_weight_grad_kernel(const float* __restrict__ slabs,
                                                                                int n, int d, float* dwq,
                                                                                float* dwk) {
    __shared__ float part[kSlabRows / 4][kSlabCols];
    const int cx = threadIdx.x % kSlabCols, ry = threadIdx.x / kSlabCols;
    const int col = blockIdx.x * kSlabCols + cx;
    float v = 0.0f;
    if (col < 2 * d) {
#pragma unroll 4
        for (int i = ry; i < n; i += kSlabRows) v += slabs[(int64_t)i * 2 * d + col];
    }
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    if (ry % 4 == 0) part[ry / 4][cx] = v;
    __syncthreads();
    if (ry == 0 && col < 2 * d) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kSlabRows / 4; ++i) s += part[i][cx];
        (col < d ? dwq : dwk)[col < d ? col : col - d] = s;
    }
}

int qk_rope_passes(int hq, int hk, int d) {
    const int lph = d <= 64 ? 4 : d <= 128 ? 8 : d <= 256 ? 16 : 32;
    const int hpw = kWave / lph;
    return (hq + hk + hpw - 1) / hpw;
}

// Streams of tokens: as many waves as run at once (the backward with norms takes 150 registers: three a SIMD),
// each with several tokens where there are many. At 8192 tokens the norms take 39 us backward with three waves a
// SIMD against 46 with four (a fourth of them in a second round), 39 with two; forward 30, 31, 35. Without norms
// 13.7 us with four over 4096 tokens, 14.1 with three.
static int qk_rope_streams(int64_t rows, int passes, bool norm) {
    const int64_t want = (norm ? 3 * kQkMaxWaves / 4 : kQkMaxWaves) / passes;
    return (int)(rows < want ? rows : (want > 0 ? want : 1));
}

int qk_rope_groups(int64_t rows, int passes, bool norm) {
    return (passes * qk_rope_streams(rows, passes, norm) + kQkWaves - 1) / kQkWaves;
}

template <int DT, int LPH, bool BWD>
static void launch_sized(const QkRopeArgs& a, bool norm, bool axes, unsigned grid, hipStream_t s) {
    if (norm && axes)
        hipLaunchKernelGGL((qk_rope_kernel<DT, LPH, true, true, BWD>), dim3(grid), dim3(kQkThreads), 0, s, a);
    else if (norm)
        hipLaunchKernelGGL((qk_rope_kernel<DT, LPH, true, false, BWD>), dim3(grid), dim3(kQkThreads), 0, s, a);
    else if (axes)
        hipLaunchKernelGGL((qk_rope_kernel<DT, LPH, false, true, BWD>), dim3(grid), dim3(kQkThreads), 0, s, a);
    else
        hipLaunchKernelGGL((qk_rope_kernel<DT, LPH, false, false, BWD>), dim3(grid), dim3(kQkThreads), 0, s, a);
}

template <int DT, bool BWD>
static void launch_typed(const QkRopeArgs& a, bool norm, bool axes, unsigned grid, hipStream_t s) {
    if (a.d <= 64)
        launch_sized<DT, 4, BWD>(a, norm, axes, grid, s);
    else if (a.d <= 128)
        launch_sized<DT, 8, BWD>(a, norm, axes, grid, s);
    else if (a.d <= 256)
        launch_sized<DT, 16, BWD>(a, norm, axes, grid, s);
    else
        launch_sized<DT, 32, BWD>(a, norm, axes, grid, s);
}

hipError_t launch_qk_rope(QkRopeArgs a, int dtype, bool norm, bool axes, bool backward, float* dwq, float* dwk,
                          hipStream_t s) {
    if (a.rows == 0) {
        // no tokens: the gradients of the weights are empty sums
        if (dwq == nullptr) return hipSuccess;
        hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((2 * a.d + kSlabCols - 1) / kSlabCols),
                           dim3(kSlabCols * kSlabRows), 0, s, a.slabs, 0, a.d, dwq, dwk);
        return hipGetLastError();
    }
    a.passes = qk_rope_passes(a.hq, a.hk, a.d);
    a.streams = qk_rope_streams(a.rows, a.passes, norm);
    const unsigned grid = (unsigned)qk_rope_groups(a.rows, a.passes, norm);
    if (dtype == DK_FP16) {
        if (backward)
            launch_typed<DK_FP16, true>(a, norm, axes, grid, s);
        else
            launch_typed<DK_FP16, false>(a, norm, axes, grid, s);
    } else {
        if (backward)
            launch_typed<DK_BF16, true>(a, norm, axes, grid, s);
        else
            launch_typed<DK_BF16, false>(a, norm, axes, grid, s);
    }
    if (dwq != nullptr)
        hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((2 * a.d + kSlabCols - 1) / kSlabCols),
                           dim3(kSlabCols * kSlabRows), 0, s, a.slabs, (int)grid, a.d, dwq, dwk);
    return hipGetLastError();
}

}  // namespace dk
