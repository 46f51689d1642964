// Dropout whose mask comes from a counter-based generator and is never stored: the forward writes
// the dropped-out inputs of up to four LoRA branches from one read of x, the backward sums the
// branches' gradients through the same masks. Each forms the mask again from (seed, offset).
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", SC 2011), key = the seed's two words, counter of columns 8 g .. 8 g + 7 of row r in branch b
// = (g, r, low word, high word of offset + b). A call gives four words, 16 bits an element: column
// 8 g + e takes half e % 2 of word e / 2 and is kept when it is >= rint(65536 p); so p is a
// multiple of 2^-16, and the kept scale is 65536 / (65536 - rint(65536 p)), the exact reciprocal of
// what is kept. The counter names the element, not the launch: strides, types and work split change
// no mask, and row r of a call is row r of any call.
//   forward:  out_b = keep_b ? x * scale_b : +0        (fp32, one rounding)
//   backward: dx = sum_b keep_b ? g_b * scale_b : 0     (fp32 in branch order, one rounding)
// A dropped element is zero whatever it held (infinities and NaN included).
//
// Bound: HBM and, nearly as much, the vector units: the generator takes 20 wide 32-bit products a group and
// branch. Sixteen bits an element instead of 32 halve its share. Two branches of [8192, 3584] fp16: forward
// 30 to 32 us (5.8 to 5.5 TB/s), backward 36 to 37 (4.9); a large copy reaches 5.2 TB/s. Three-input exclusive ors and the
// row by a multiplication instead of a division took 2 to 3 us off each. One thread a group keeps every load
// of a wave contiguous and the device full.
#include "elem.h"

namespace dk {

constexpr int kDropoutThreads = 256;

struct Philox {
    uint32_t w[4];
};

__device__ __forceinline__ Philox philox10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                           uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), c1, k0, 0x96);  // a ^ b ^ c
        c1 = (uint32_t)b;
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), c3, k1, 0x96);
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Philox{{c0, c1, c2, c3}};
}

// the kept elements of a group times scale, zeros elsewhere
__device__ __forceinline__ float8_t drop8(float8_t v, const Philox& p, uint32_t thr, float scale) {
    float8_t o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t bits = e & 1 ? p.w[e / 2] >> 16 : p.w[e / 2] & 0xFFFFu;
        o[e] = bits >= thr ? v[e] * scale : 0.0f;
    }
    return o;
}

template <int DT>
__device__ __forceinline__ float8_t load_group(const void* row, uint32_t col, uint32_t width) {
    const typename Elem<DT>::type* p = (const typename Elem<DT>::type*)row + col;
    if (col + 8 <= width) return load8<DT>(p);
    float8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < width) v[e] = (float)p[e];
    return v;
}

template <int DT>
__device__ __forceinline__ void store_group(void* row, uint32_t col, uint32_t width, float8_t v) {
    typename Elem<DT>::type* p = (typename Elem<DT>::type*)row + col;
    if (col + 8 <= width) {
        store8<DT>(p, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < width) store1<DT>(p + e, v[e]);
}

// NB branches (0: a.nb of them). One thread takes one group of eight columns of one row.
template <int IN, int OUT, int NB, bool BWD>
__global__ __launch_bounds__(kDropoutThreads) void dropout_kernel(const DropoutArgs a) {
    const uint32_t i = blockIdx.x * kDropoutThreads + threadIdx.x;
    if (i >= a.items) return;
    // i / groups by a multiplication (exact for i < 2^31)
    const uint32_t row = a.groups == 1 ? i : __umulhi(i, a.div_mul) >> a.div_shift, g = i - row * a.groups;
    const uint64_t seed = (uint64_t)a.rng[0], offset = (uint64_t)a.rng[1];
    const auto bits = [&](int b) {
        const uint64_t o = offset + (uint64_t)b;
        return philox10(g, row, (uint32_t)o, (uint32_t)(o >> 32), (uint32_t)seed, (uint32_t)(seed >> 32));
    };
    const auto in = [&](int b) {
        return (const char*)a.in[b] + (int64_t)row * a.ld_in[b] * elem_bytes(IN);
    };
    const auto out = [&](int b) { return (char*)a.out[b] + (int64_t)row * a.ld_out[b] * elem_bytes(OUT); };
    if constexpr (!BWD) {
        const float8_t x = load_group<IN>(in(0), 8 * g, a.width);
        const auto branch = [&](int b) {
            store_group<OUT>(out(b), 8 * g, a.width, drop8(x, bits(b), a.thr[b], a.scale[b]));
        };
        if constexpr (NB != 0) {
#pragma unroll
            for (int b = 0; b < NB; ++b) branch(b);
        } else {
            for (int b = 0; b < a.nb; ++b) branch(b);
        }
    } else {
        float8_t sum = {0, 0, 0, 0, 0, 0, 0, 0};
        if constexpr (NB != 0) {
            // every branch's load in flight before the first mask
            float8_t v[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) v[b] = load_group<IN>(in(b), 8 * g, a.width);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float8_t d = drop8(v[b], bits(b), a.thr[b], a.scale[b]);
                sum = b == 0 ? d : sum + d;
            }
        } else {
            for (int b = 0; b < a.nb; ++b) {
                if (a.in[b] == nullptr) continue;  // a branch without a gradient
                sum = sum + drop8(load_group<IN>(in(b), 8 * g, a.width), bits(b), a.thr[b], a.scale[b]);
            }
        }
        store_group<OUT>(out(0), 8 * g, a.width, sum);
    }
}

template <int IN, int OUT, bool BWD>
static void launch_typed(const DropoutArgs& a, unsigned grid, hipStream_t s) {
    bool whole = true;
    if (BWD)
        for (int b = 0; b < a.nb; ++b) whole = whole && a.in[b] != nullptr;
    if (a.nb == 1 && whole)
        hipLaunchKernelGGL((dropout_kernel<IN, OUT, 1, BWD>), dim3(grid), dim3(kDropoutThreads), 0, s, a);
    else if (a.nb == 2 && whole)
        hipLaunchKernelGGL((dropout_kernel<IN, OUT, 2, BWD>), dim3(grid), dim3(kDropoutThreads), 0, s, a);
    else
        hipLaunchKernelGGL((dropout_kernel<IN, OUT, 0, BWD>), dim3(grid), dim3(kDropoutThreads), 0, s, a);
}

template <bool BWD>
static void launch_way(const DropoutArgs& a, int in, int out, unsigned grid, hipStream_t s) {
    if (in == DK_FP32) {
        if (out == DK_FP32) launch_typed<DK_FP32, DK_FP32, BWD>(a, grid, s);
        else if (out == DK_FP16) launch_typed<DK_FP32, DK_FP16, BWD>(a, grid, s);
        else launch_typed<DK_FP32, DK_BF16, BWD>(a, grid, s);
    } else if (in == DK_FP16) {
        if (out == DK_FP32) launch_typed<DK_FP16, DK_FP32, BWD>(a, grid, s);
        else launch_typed<DK_FP16, DK_FP16, BWD>(a, grid, s);
    } else {
        if (out == DK_FP32) launch_typed<DK_BF16, DK_FP32, BWD>(a, grid, s);
        else launch_typed<DK_BF16, DK_BF16, BWD>(a, grid, s);
    }
}

hipError_t launch_dropout(DropoutArgs a, int in_dtype, int out_dtype, bool backward, hipStream_t s) {
    if (a.items == 0) return hipSuccess;
    // i / d = (i m) >> (31 + l), l = ceil(log2 d), m = floor(2^(31 + l) / d) + 1: m d exceeds 2^(31 + l) by
    // at most d <= 2^l, which times i < 2^31 stays below 2^(31 + l)
    int l = 0;
    while ((uint64_t(1) << l) < a.groups) ++l;
    if (a.groups > 1) {
        a.div_mul = (uint32_t)((uint64_t(1) << (31 + l)) / a.groups + 1);
        a.div_shift = (uint32_t)(l - 1);
    }
    const unsigned grid = (unsigned)(((uint64_t)a.items + kDropoutThreads - 1) / kDropoutThreads);
    if (backward)
        launch_way<true>(a, in_dtype, out_dtype, grid, s);
    else
        launch_way<false>(a, in_dtype, out_dtype, grid, s);
    return hipGetLastError();
}

}  // namespace dk
