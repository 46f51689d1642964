// Rotary positions of q and k heads: the first R elements of each head turn, the other D - R pass through. With angle
// t_j = position * inv_freq[j], c_j = factor cos t_j, s_j = factor sin t_j, j < R / 2, the elements (a, b) of pair j --
// (x[j], x[j + R / 2]) in halves, (x[2 j], x[2 j + 1]) in pairs -- become
//   forward: (a c - b s, b c + a s)        back: (a c + b s, b c - a s)
// in fp32, one rounding at the end. Token-major in and head-major out, or, back, the other way round.
//
// Angles are formed in turns as 64-bit fixed-point fractions (turn_fraction), so that whole turns drop out exactly, and reach
// sincospif as fp32 half turns: within 2^-24 turns at positions below 2^28, where an fp32 product of position and frequency
// is off by 2^-5 radians at 2^20 already.
// A work-group takes a few tokens, forms each of their R / 2 cosines and sines once, in LDS, and turns all heads with
// them; a thread has one or two items in flight. An item is 16 elements, two 16-byte loads (halves with R and D
// multiples of 16: both elements of eight pairs), or eight: with pairs whole, with halves of any even R and their
// partners loaded beside them (lines that the work-group reads anyway). Sizes of D that are no multiple of eight go
// pair by pair.
//
// Bound: HBM (q and k in and out): 8192 tokens of 28 + 4 heads of 128, bf16, 26.7 us either way with q and k from memory
// (5.0 TB/s; a large copy reaches 5.2). Three sequences of 683 tokens, 9 + 3 heads of 80, a quarter turned, 7.4 us and 16
// single tokens 3.7: a launch and two memory round trips. The tables' reads in halves use some banks twice (LDS busy
// 41% of the time): a layout without that was no faster (27.2 us).
#include "elem.h"

namespace dk {

constexpr int kScaledThreads = 256;

enum { HALF16, PAIRS8, HALF8, SINGLE };

// elements an item covers in a head, SINGLE: a pair or an element that passes through
__device__ __host__ constexpr int items_a_head(int mode, int d, int r) {
    return mode == HALF16 ? d / 16 : mode == SINGLE ? d - r / 2 : d / 8;
}

template <int DT, int MODE, int U>
__global__ __launch_bounds__(kScaledThreads) void scaled_rope_kernel(const ScaledRopeArgs a) {
    typedef typename Elem<DT>::type elem_t;
    typedef typename Elem<DT>::vec vec_t;
    extern __shared__ __attribute__((aligned(16))) float2_t trig[];  // [tokens of the work-group][R / 2]
    const int half = a.r / 2, per = items_a_head(MODE, a.d, a.r);
    const uint32_t first = blockIdx.x * a.tpw, count = min((uint32_t)a.tpw, a.rows - first);
    const uint32_t total = (uint32_t)(a.hq + a.hk) * count * per;

    // an item's place: its tensor's elements in and out, its token of the work-group, its index in the head
    struct Place {
        const elem_t* in;
        elem_t* out;
        int token, item;
    };
    const auto place = [&](uint32_t i) {
        Place p;
        const uint32_t rest = i / per;
        p.item = (int)(i - rest * per);
        const uint32_t slot = rest / count;
        p.token = (int)(rest - slot * count);
        const bool isq = slot < (uint32_t)a.hq;
        const int64_t head = isq ? slot : slot - a.hq;
        const uint32_t row = first + p.token, b = row / a.tokens, t = row - b * a.tokens;
        const int64_t* const si = isq ? a.q_in : a.k_in;
        const int64_t* const so = isq ? a.q_st : a.k_st;
        p.in = (const elem_t*)(isq ? a.q : a.k) + b * si[0] + t * si[1] + head * si[2];
        p.out = (elem_t*)(isq ? a.oq : a.ok) + b * so[0] + t * so[1] + head * so[2];
        return p;
    };
    // where an item's first and second eight elements start, and whether and where the second belong to the first
    const auto at0 = [&](int item) {
        if (MODE == HALF16) return 16 * item < a.r ? 8 * item : 16 * item;
        return 8 * item;
    };
    const auto at1 = [&](int item) {
        const int c = 8 * item;
        if (MODE == HALF16) return 16 * item < a.r ? half + c : 16 * item + 8;
        // HALF8: the partners of eight elements of one half; a chunk across an edge has them read one by one
        return c + 8 <= half ? c + half : c >= half && c + 8 <= a.r ? c - half : c;
    };

    Place p[U];
    vec_t va[U], vb[U];
    const auto fetch = [&](uint32_t base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            p[u] = place(min(base + u * kScaledThreads, total - 1));
            if constexpr (MODE != SINGLE) va[u] = load8_raw<DT>(p[u].in + at0(p[u].item));
            if constexpr (MODE == HALF16 || MODE == HALF8) vb[u] = load8_raw<DT>(p[u].in + at1(p[u].item));
        }
    };
    fetch(threadIdx.x);

    for (uint32_t i = threadIdx.x; i < count * half; i += kScaledThreads) {
        const uint32_t tok = i / half, j = i - tok * half, row = first + tok, b = row / a.tokens, t = row - b * a.tokens;
        const int64_t at = (int64_t)b * a.pos_batch + t;
        const int64_t pos = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
        const int32_t turn = (int32_t)((turn_fraction(a.inv_freq[j]) * (uint64_t)pos) >> 32);
        float s, c;
        sincospif((float)turn * 4.656612873077393e-10f, &s, &c);  // 2^-31 half turns
        trig[i] = float2_t{c * a.factor, s * a.sin_factor};
    }
    __syncthreads();

    for (uint32_t base = threadIdx.x; base < total; base += U * kScaledThreads) {
        if (base != threadIdx.x) fetch(base);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float2_t* const cs = trig + p[u].token * half;
            const int item = p[u].item;
            elem_t* const out = p[u].out;
            if constexpr (MODE == HALF16) {
                if (16 * item < a.r) {
                    const float8_t x = widen8<DT>(va[u]), y = widen8<DT>(vb[u]);
                    float8_t c, s;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        c[e] = cs[8 * item + e].x;
                        s[e] = cs[8 * item + e].y;
                    }
                    store8<DT>(out + at0(item), x * c - y * s);
                    store8<DT>(out + at1(item), y * c + x * s);
                } else {
                    *(typename Elem<DT>::loose*)(out + at0(item)) = va[u];
                    *(typename Elem<DT>::loose*)(out + at1(item)) = vb[u];
                }
            } else if constexpr (MODE == PAIRS8) {
                const float8_t x = widen8<DT>(va[u]);
                vec_t o = va[u];
                if (8 * item < a.r) {
                    float8_t y;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        // (past R within the last chunk: its last pair's table entry, not used)
                        const float2_t c = cs[min(4 * item + e / 2, half - 1)];
                        y[e] = x[e] * c.x - x[e + 1] * c.y;
                        y[e + 1] = x[e + 1] * c.x + x[e] * c.y;
                    }
                    const int left = a.r - 8 * item;
                    if (left >= 8) {
                        store8<DT>(out + 8 * item, y);
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float f = y[e];
                        asm("" : "+v"(f));
                        o[e] = e < left ? (elem_t)f : o[e];
                    }
                }
                *(typename Elem<DT>::loose*)(out + 8 * item) = o;
            } else if constexpr (MODE == HALF8) {
                const float8_t x = widen8<DT>(va[u]);
                float8_t y = widen8<DT>(vb[u]);
                const int c0 = 8 * item;
                const bool low = c0 + 8 <= half, high = c0 >= half && c0 + 8 <= a.r;
                if (!low && !high && c0 < a.r) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int at = c0 + e;
                        if (at < a.r) y[e] = (float)p[u].in[at < half ? at + half : at - half];
                    }
                }
                vec_t o = va[u];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = c0 + e, j = at < half ? at : at - half;
                    if (at < a.r) {
                        const float2_t c = cs[j];
                        float f = at < half ? x[e] * c.x - y[e] * c.y : x[e] * c.x + y[e] * c.y;
                        asm("" : "+v"(f));
                        o[e] = (elem_t)f;
                    }
                }
                *(typename Elem<DT>::loose*)(out + c0) = o;
            } else {
                const elem_t* const in = p[u].in;
                if (item < half) {
                    const int i0 = a.pairs ? 2 * item : item, i1 = a.pairs ? 2 * item + 1 : half + item;
                    const float x = (float)in[i0], y = (float)in[i1];
                    const float2_t c = cs[item];
                    store1<DT>(out + i0, x * c.x - y * c.y);
                    store1<DT>(out + i1, y * c.x + x * c.y);
                } else {
                    const int at = half + item;
                    out[at] = in[at];
                }
            }
        }
    }
}

template <int DT, int MODE>
static void launch_items(const ScaledRopeArgs& a, bool many, hipStream_t s) {
    const dim3 grid((a.rows + a.tpw - 1) / a.tpw), threads(kScaledThreads);
    const size_t lds = (size_t)a.tpw * (a.r / 2) * sizeof(float2_t);
    if (many)
        hipLaunchKernelGGL((scaled_rope_kernel<DT, MODE, 2>), grid, threads, lds, s, a);
    else
        hipLaunchKernelGGL((scaled_rope_kernel<DT, MODE, 1>), grid, threads, lds, s, a);
}

template <int DT>
static void launch_mode(const ScaledRopeArgs& a, int mode, bool many, hipStream_t s) {
    switch (mode) {
        case HALF16: launch_items<DT, HALF16>(a, many, s); break;
        case PAIRS8: launch_items<DT, PAIRS8>(a, many, s); break;
        case HALF8: launch_items<DT, HALF8>(a, many, s); break;
        default: launch_items<DT, SINGLE>(a, many, s);
    }
}

hipError_t launch_scaled_rope(ScaledRopeArgs a, int dtype, hipStream_t s) {
    const int mode = a.d % 8 != 0                                ? SINGLE
                     : a.pairs                                   ? PAIRS8
                     : a.d % 16 == 0 && a.r % 16 == 0 && a.r > 0 ? HALF16
                                                                 : HALF8;
    // Tokens a work-group: about two items a thread where the tokens are enough for two work-groups a CU, else one
    // token, so that few tokens spread over the CUs; at most 32 KB of tables. (8192 tokens of 28 + 4 heads of 128, bf16: 26.7
    // us; four items a thread 30.9, of which two in flight at a time 28.5, eight items 30.8.)
    const int64_t items = (int64_t)(a.hq + a.hk) * items_a_head(mode, a.d, a.r);
    const int64_t table = (int64_t)(a.r > 0 ? a.r / 2 : 1) * (int64_t)sizeof(float2_t);
    int64_t tpw = 2 * kScaledThreads / items;
    tpw = tpw < 1 ? 1 : tpw > 16 ? 16 : tpw;
    while (tpw > 1 && (a.rows < 512 * tpw || tpw * table > 32768)) tpw /= 2;
    a.tpw = (int32_t)tpw;
    const bool many = tpw * items > kScaledThreads;
    if (dtype == DK_FP16)
        launch_mode<DK_FP16>(a, mode, many, s);
    else
        launch_mode<DK_BF16>(a, mode, many, s);
    return hipGetLastError();
}

}  // namespace dk
