// Linear layers whose weight holds 4-bit integers with a scale and a zero point for every group of columns of a row:
//   W[n, k] = (code[n, k] - zero[n, k / group]) scale[n, k / group]
//   forward   y[m, n]  = sum over groups g of scale[n, g] (sum over k in g of x[m, k] (code[n, k] - zero[n, g])) + bias[n]
//   backward  dx[m, k] = sum over n of dy[m, n] W[n, k]
// on 16x16x32 MFMAs of the activations' type with fp32 sums. The forward's matrix operands are exact, code - zero a small
// integer, and the scale is applied to a group's fp32 sum: nothing is rounded but the sums and the output. The
// backward sums over rows, each with its own scale, so there W is rounded once to 16 bits, as the matrix cores take it (at
// most half a step of the type a weight, of alternating sign along a sum).
//
// Layout of a row: blocks of 128 columns in 64 bytes, so that a lane's 16 bytes are its operands of four MFMAs as they lie:
// dword 4 q + j of a block holds columns 32 j + 8 q + 0 .. 7, column 2 i of those in bits 4 i, column 2 i + 1 in bits
// 16 + 4 i (a shift and a mask leave a pair in the halves of a register). In each MFMA lane l = 16 q + r holds k
// = 8 q + 0 .. 7 of row r of its operand. `meta` holds a group's scale (low 16 bits) and zero point (next byte).
// From pairs to operands, fp16: 0x6400 | q is 1024 + q, 0x6400 | 16 q is 1024 + 16 q, and one packed subtraction or
// multiply-add leaves q - zero, exactly. bf16: 0x4180 | 8 q is 16 + q; there is no packed bf16 arithmetic, so 16 + zero
// times the sum of x, from one more MFMA, is taken off the group's sum.
#include "elem.h"
#include "gemm_common.h"

namespace dk {

constexpr int kI4Block = 128;  // columns of a block

template <int DT>
struct I4;
template <>
struct I4<DK_FP16> {
    typedef half8_t vec;
    static __device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float scale(uint32_t meta) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)meta);
    }
};
template <>
struct I4<DK_BF16> {
    typedef bf16x8_t vec;
    static __device__ __forceinline__ float4_t mfma(bf16x8_t a, bf16x8_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float scale(uint32_t meta) { return __builtin_bit_cast(float, meta << 16); }
};

__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) { return (v & mask) | bits; }

__device__ __forceinline__ float zero_of(uint32_t meta) { return (float)((meta >> 16) & 0xFF); }

// scale of either 16-bit type
__device__ __forceinline__ float scale_of(uint32_t meta, int scale_dtype) {
    return scale_dtype == DK_BF16 ? I4<DK_BF16>::scale(meta) : I4<DK_FP16>::scale(meta);
}

// pairs of zero-point constants of a row for the forward: fp16 -(1024 + zero) and -(64 + zero); bf16 unused
struct ZeroF16 {
    half2_t whole, part;
    __device__ __forceinline__ void set(uint32_t meta) {
        const _Float16 z = (_Float16)zero_of(meta);
        const _Float16 a = (_Float16)-1024.0f - z, b = (_Float16)-64.0f - z;
        whole = half2_t{a, a};
        part = half2_t{b, b};
    }
};

// eight operands of a dword: fp16 code - zero, bf16 16 + code
template <int DT>
__device__ __forceinline__ typename I4<DT>::vec unpack8(uint32_t d, const ZeroF16& z) {
    u32x4_t o;
    if constexpr (DT == DK_FP16) {
        const uint32_t h = d >> 8;
        const half2_t sixteenth = half2_t{(_Float16)0.0625f, (_Float16)0.0625f};
        const auto even = [&](uint32_t v) {
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, and_or(v, 0x000F000Fu, 0x64006400u)) + z.whole);
        };
        const auto odd = [&](uint32_t v) {
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, and_or(v, 0x00F000F0u, 0x64006400u)),
                                                                          sixteenth, z.part));
        };
        o = u32x4_t{even(d), odd(d), even(h), odd(h)};
    } else {
        o = u32x4_t{and_or(d << 3, 0x00780078u, 0x41804180u), and_or(d >> 1, 0x00780078u, 0x41804180u),
                    and_or(d >> 5, 0x00780078u, 0x41804180u), and_or(d >> 9, 0x00780078u, 0x41804180u)};
    }
    return __builtin_bit_cast(typename I4<DT>::vec, o);
}

// group of the 32 columns that begin at 32 unit
__device__ __forceinline__ uint32_t group_at(const Int4Args& a, uint32_t unit) {
    return a.group_units == 1 ? unit : __umulhi(unit, a.group_mul);
}

__device__ __forceinline__ void store_out(const Int4Args& a, int64_t at, float v) {
    asm("" : "+v"(v));
    if (a.y_dtype == DK_FP32)
        ((float*)a.y)[at] = v;
    else if (a.y_dtype == DK_BF16)
        ((__bf16*)a.y)[at] = (__bf16)v;
    else
        ((_Float16*)a.y)[at] = (_Float16)v;
}

// ---- forward, few tokens -------------------------------------------------------------------------
// A work-group takes 16 rows of the weight and 16 C tokens; its NW waves share the columns, each streaming its blocks
// to registers (P blocks in flight), and join their sums through LDS. GJ: the 32-column units a scale is
// constant over (4, 2 or 1).
template <int DT, int C, int GJ, int NW, int P>
__global__ __launch_bounds__(64 * NW) void int4_few_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    constexpr int UNITS = 4 / GJ;
    __shared__ float sums[NW][C * 4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * C;
    const int rows = min(16, a.n - n0), toks = min(16 * C, a.m - m0);
    const int per = (a.blocks + NW - 1) / NW, b0 = wave * per, b1 = min(a.blocks, b0 + per);

    const rsrc_t wr = make_rsrc(a.w + (int64_t)n0 * a.ldw, (uint32_t)(rows * a.ldw));
    const rsrc_t mr = make_rsrc(a.meta + (int64_t)n0 * a.groups, (uint32_t)(rows * a.groups * 4));
    const rsrc_t xr = make_rsrc((const uint16_t*)a.x + (int64_t)m0 * a.ldx, (uint32_t)(((toks - 1) * a.ldx + a.x_cols) * 2));
    const uint32_t w_at = r * (uint32_t)a.ldw + 16 * q, m_at = r * (uint32_t)a.groups * 4;
    uint32_t x_at[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x_at[c] = off_if(16 * c + r < toks, (16 * c + r) * (uint32_t)a.ldx * 2 + 16 * q);

    struct Stage {
        u32x4_t w;
        uint32_t meta[UNITS];
        u32x4_t x[C][4];
    };
    Stage st[P];
    const auto fetch = [&](Stage& s, int b) {
        const bool live = b < b1;
        s.w = bload128(wr, off_if(live, w_at + 64 * (uint32_t)b));
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t unit = 4 * b + GJ * u;
            // (a last block's units past k have no group: they read the last one's, for x of zeros)
            const uint32_t g = min(group_at(a, unit), (uint32_t)a.groups - 1);
            s.meta[u] = __builtin_amdgcn_raw_buffer_load_b32(mr, (int)off_if(live, m_at + 4 * g), 0, 0);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = kI4Block * b + 32 * j + 8 * q;
                s.x[c][j] = bload128(xr, off_if(live && col < a.x_cols, x_at[c] + 256 * (uint32_t)b + 64 * j));
            }
    };
    float4_t acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = float4_t{};
    const auto compute = [&](const Stage& s) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t meta = s.meta[u];
            ZeroF16 z;
            vec taken;
            if constexpr (DT == DK_FP16) {
                z.set(meta);
            } else {
                const __bf16 t = (__bf16)(-16.0f - zero_of(meta));
                taken = vec{t, t, t, t, t, t, t, t};
            }
            float4_t t[C];
#pragma unroll
            for (int c = 0; c < C; ++c) t[c] = float4_t{};
#pragma unroll
            for (int j = GJ * u; j < GJ * (u + 1); ++j) {
                const vec w = unpack8<DT>(s.w[j], z);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const vec x = __builtin_bit_cast(vec, s.x[c][j]);
                    t[c] = I4<DT>::mfma(x, w, t[c]);
                    if constexpr (DT == DK_BF16) t[c] = I4<DT>::mfma(x, taken, t[c]);
                }
            }
            const float scale = scale_of(meta, a.scale_dtype);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_fmaf(t[c][i], scale, acc[c][i]);
        }
    };
#pragma unroll
    for (int p = 0; p < P; ++p) fetch(st[p], b0 + p);
    for (int b = b0; b < b1; b += P) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            compute(st[p]);
            fetch(st[p], b + p + P);
        }
    }

    // lane: row n0 + r, tokens m0 + 16 c + 4 q + i
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][4 * c + i][lane] = acc[c][i];
    __syncthreads();
    for (int e = threadIdx.x; e < C * 4 * 64; e += 64 * NW) {
        const int slot = e >> 6, l = e & 63;
        const int m = m0 + 16 * (slot >> 2) + 4 * (l >> 4) + (slot & 3), n = n0 + (l & 15);
        if (m >= a.m || n >= a.n) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += sums[w][slot][l];
        if (a.bias != nullptr) v += load_any(a.bias, a.bias_dtype, n);
        store_out(a, (int64_t)m * a.ldy + n, v);
    }
}

// ---- forward, many tokens ------------------------------------------------------------------------
// Tiles of 128 tokens by 256 rows of the weight, eight waves of 64 by 64. The tokens' block of 128 columns goes to LDS
// (two stages, 16-byte chunks permuted by row against bank conflicts), the weight to registers, a block ahead.
constexpr int kI4TileM = 128, kI4TileN = 256, kI4Waves = 8;
constexpr int kI4StageBytes = kI4TileM * kI4Block * 2;

// consecutive tiles on one XCD, token tiles fastest within bands of eight (the same order as the 8-bit products)
__device__ __forceinline__ void tile_of(const Int4Args& a, int& m_tile, int& n_tile, int& split) {
    const int per = a.m_tiles * a.n_tiles, nwg = per * a.splits;
    const int xcd = blockIdx.x & 7, r8 = nwg & 7;
    const int L = xcd * (nwg >> 3) + min(xcd, r8) + (blockIdx.x >> 3);
    split = L / per;
    const int tile = L - split * per;
    const int band = tile / (8 * a.n_tiles), in = tile - band * 8 * a.n_tiles;
    const int rows = min(8, a.m_tiles - 8 * band);
    m_tile = 8 * band + in % rows;
    n_tile = in / rows;
}

// 16 rows of `cols` outputs a wave holds through LDS leave as 16-byte pieces
template <int DT>
__device__ __forceinline__ void put_row8(const Int4Args& a, const uint16_t* from, int64_t at, int left) {
    typedef typename Elem<DT>::type E;
    if (left >= 8) {
        *(typename Elem<DT>::loose*)((E*)a.y + at) = *(const typename Elem<DT>::vec*)from;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) ((E*)a.y)[at + e] = ((const E*)from)[e];
    }
}

template <int DT, int GJ>
__global__ __launch_bounds__(64 * kI4Waves, 2) void int4_tile_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    constexpr int UNITS = 4 / GJ, R = 4, C = 4, XLOADS = kI4StageBytes / 1024 / kI4Waves;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    int mt, nt, split;
    tile_of(a, mt, nt, split);
    const int m0 = mt * kI4TileM, n0 = nt * kI4TileN;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int b0 = split * a.blocks_per_split, steps = min(a.blocks_per_split, a.blocks - b0);

    const int rows = min(64, a.n - n0 - wn), toks = min(kI4TileM, a.m - m0);
    const rsrc_t wr = make_rsrc(a.w + (int64_t)(n0 + wn) * a.ldw, rows > 0 ? (uint32_t)(rows * a.ldw) : 0u);
    const rsrc_t mr = make_rsrc(a.meta + (int64_t)(n0 + wn) * a.groups, rows > 0 ? (uint32_t)(rows * a.groups * 4) : 0u);
    const rsrc_t xr = make_rsrc((const uint16_t*)a.x + (int64_t)m0 * a.ldx, (uint32_t)(((toks - 1) * a.ldx + a.x_cols) * 2));
    uint32_t x_at[XLOADS];
    int x_col[XLOADS];
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
        const int row = 4 * (wave * XLOADS + i) + (lane >> 4);
        x_col[i] = 8 * ((lane & 15) ^ (row & 15));
        x_at[i] = off_if(row < toks, (row * (uint32_t)a.ldx + x_col[i]) * 2);
    }
    const auto fetch_x = [&](int t) {
        const int k0 = (b0 + t) * kI4Block;
#pragma unroll
        for (int i = 0; i < XLOADS; ++i)
            bload128_lds(xr, smem + (t & 1) * kI4StageBytes + 1024 * (wave * XLOADS + i),
                         off_if(t < steps && k0 + x_col[i] < a.x_cols, x_at[i] + 2 * (uint32_t)k0));
    };
    struct Weights {
        u32x4_t w[R];
        uint32_t meta[R][UNITS];
    };
    const auto fetch_w = [&](Weights& f, int t) {
        const uint32_t b = b0 + t;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint32_t row = 16 * i + r;
            f.w[i] = bload128(wr, off_if(t < steps, row * (uint32_t)a.ldw + 16 * q + 64 * b));
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const uint32_t g = min(group_at(a, 4 * b + GJ * u), (uint32_t)a.groups - 1);
                f.meta[i][u] = __builtin_amdgcn_raw_buffer_load_b32(
                    mr, (int)off_if(t < steps, (row * (uint32_t)a.groups + g) * 4), 0, 0);
            }
        }
    };

    float4_t acc[R][C];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[i][c] = float4_t{};
    const vec ones = __builtin_bit_cast(vec, u32x4_t{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});  // bf16

    Weights f;
    fetch_w(f, 0);
    fetch_x(0);
    for (int t = 0; t < steps; ++t) {
        wait_vmcnt<0>();
        lds_barrier();  // the stage is whole, and every wave has read the one before it
        const Weights now = f;
        fetch_w(f, t + 1);
        fetch_x(t + 1);
        const uint8_t* const stage = smem + (t & 1) * kI4StageBytes;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            float4_t s[R][C], xs[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                xs[c] = float4_t{};
#pragma unroll
                for (int i = 0; i < R; ++i) s[i][c] = float4_t{};
            }
            ZeroF16 z[R];
            if constexpr (DT == DK_FP16) {
#pragma unroll
                for (int i = 0; i < R; ++i) z[i].set(now.meta[i][u]);
            }
#pragma unroll
            for (int j = GJ * u; j < GJ * (u + 1); ++j) {
                vec x[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int row = wm + 16 * c + r;
                    x[c] = *(const vec*)(stage + row * 256 + 16 * ((4 * j + q) ^ r));
                }
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const vec w = unpack8<DT>(now.w[i][j], z[i]);
#pragma unroll
                    for (int c = 0; c < C; ++c) s[i][c] = I4<DT>::mfma(x[c], w, s[i][c]);
                }
                if constexpr (DT == DK_BF16) {
#pragma unroll
                    for (int c = 0; c < C; ++c) xs[c] = I4<DT>::mfma(x[c], ones, xs[c]);
                }
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float scale = scale_of(now.meta[i][u], a.scale_dtype);
                const float taken = -16.0f - zero_of(now.meta[i][u]);
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = s[i][c][e];
                        if constexpr (DT == DK_BF16) v = __builtin_fmaf(taken, xs[c][e], v);
                        acc[i][c][e] = __builtin_fmaf(v, scale, acc[i][c][e]);
                    }
            }
        }
    }
    wait_vmcnt<0>();
    lds_barrier();

    // lane: row wn + 16 i + r of the weight, tokens wm + 16 c + 4 q + e
    if (a.splits > 1 || a.y_dtype == DK_FP32) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int n = n0 + wn + 16 * i + r;
            if (n >= a.n) continue;
            const float bias = a.splits == 1 && a.bias != nullptr ? load_any(a.bias, a.bias_dtype, n) : 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = m0 + wm + 16 * c + 4 * q + e;
                    if (m >= a.m) continue;
                    if (a.splits > 1)
                        a.partials[split * a.slab + (int64_t)m * a.n + n] = acc[i][c][e];
                    else
                        ((float*)a.y)[(int64_t)m * a.ldy + n] = acc[i][c][e] + bias;
                }
        }
        return;
    }
    uint16_t* const mine = (uint16_t*)smem + wave * 64 * 72;  // rows of 64 outputs, padded
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int n = n0 + wn + 16 * i + r;
        const float bias = a.bias != nullptr && n < a.n ? load_any(a.bias, a.bias_dtype, n) : 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) store1<DT>(mine + (16 * c + 4 * q + e) * 72 + 16 * i + r, acc[i][c][e] + bias);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        const int row = 8 * s + (lane >> 3), m = m0 + wm + row, n = n0 + wn + 8 * (lane & 7);
        if (m < a.m && n < a.n) put_row8<DT>(a, mine + row * 72 + 8 * (lane & 7), (int64_t)m * a.ldy + n, a.n - n);
    }
}

// ---- backward ------------------------------------------------------------------------------------
// Tiles of 32 C tokens by 256 columns, four waves of 16 C by 128. A lane holds one dword of eight columns of each of
// eight rows; halves of two rows' dwords joined in one register unpack to pairs along the rows, MFMA j's operand
// for column j of every lane's dword, so that the weight needs no other layout than the forward's. Its sums come out eight
// columns a lane. Rows' scales and zero points go through LDS, a block of 128 rows ahead, as do dy's columns.
constexpr int kI4BackN = 128, kI4BackCols = 256, kI4BackUnits = kI4BackCols / 32;

template <int DT>
struct BackMeta;  // of the eight rows of a lane and step
template <>
struct BackMeta<DK_FP16> {
    half8_t scale, zero;  // scale, -(1024 + zero)
    typedef _Float16 elem;
    static constexpr int bytes = 2;
};
template <>
struct BackMeta<DK_BF16> {
    float8_t scale, zero;  // scale, -(16 + zero) scale
    typedef float elem;
    static constexpr int bytes = 4;
};

// MFMA operands of one pair of rows for the eight columns of their dwords: two weights a register
template <int DT>
__device__ __forceinline__ void weights_of_pair(uint32_t d0, uint32_t d1, const BackMeta<DT>& m, int pair, uint32_t (&o)[8]) {
    const uint32_t even = perm_lo(d0, d1), odd = perm_hi(d0, d1);  // columns 0 2 4 6, columns 1 3 5 7
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t v = h ? odd : even;
            if constexpr (DT == DK_FP16) {
                half2_t w = __builtin_bit_cast(half2_t, and_or(v >> (4 * i), 0x000F000Fu, 0x64006400u));
                w = w + half2_t{m.zero[2 * pair], m.zero[2 * pair + 1]};
                w = w * half2_t{m.scale[2 * pair], m.scale[2 * pair + 1]};
                o[2 * i + h] = __builtin_bit_cast(uint32_t, w);
            } else {
                const uint32_t w = and_or(i == 0 ? v << 3 : v >> (4 * i - 3), 0x00780078u, 0x41804180u);
                typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
                const float2_t f = float2_t{__builtin_fmaf(__builtin_bit_cast(float, w << 16), m.scale[2 * pair], m.zero[2 * pair]),
                                            __builtin_fmaf(__builtin_bit_cast(float, w & 0xFFFF0000u), m.scale[2 * pair + 1],
                                                           m.zero[2 * pair + 1])};
                o[2 * i + h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
            }
        }
    }
}

template <int DT, int C>
constexpr size_t int4_back_lds() {
    return 2 * (32 * C * kI4BackN * 2 + 2 * kI4BackUnits * kI4BackN * BackMeta<DT>::bytes);
}

template <int DT, int C>
__global__ __launch_bounds__(256, 2) void int4_back_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    typedef typename BackMeta<DT>::elem meta_t;
    constexpr int TM = 32 * C, XBYTES = TM * kI4BackN * 2, XLOADS = XBYTES / 4096, TABLE = kI4BackUnits * kI4BackN;
    constexpr int STAGE = XBYTES + 2 * TABLE * (int)sizeof(meta_t), METAS = TABLE / 256;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    int mt, kt, split;
    tile_of(a, mt, kt, split);
    const int m0 = mt * TM, k0 = kt * kI4BackCols;
    const int wm = (wave & 1) * 16 * C, wk = (wave >> 1) * 128;
    const int b0 = split * a.blocks_per_split, steps = min(a.blocks_per_split, a.blocks - b0);  // of 128 rows

    const int toks = min(TM, a.m - m0);
    const rsrc_t xr = make_rsrc((const uint16_t*)a.x + (int64_t)m0 * a.ldx, (uint32_t)(((toks - 1) * a.ldx + a.x_cols) * 2));
    uint32_t x_at[XLOADS];
    int x_col[XLOADS];
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
        const int row = 4 * (wave * XLOADS + i) + (lane >> 4);
        x_col[i] = 8 * ((lane & 15) ^ (row & 15));
        x_at[i] = off_if(row < toks, (row * (uint32_t)a.ldx + x_col[i]) * 2);
    }
    const auto fetch_x = [&](int t) {
        const int n0 = (b0 + t) * kI4BackN;
#pragma unroll
        for (int i = 0; i < XLOADS; ++i)
            bload128_lds(xr, smem + (t & 1) * STAGE + 1024 * (wave * XLOADS + i),
                         off_if(t < steps && n0 + x_col[i] < a.x_cols, x_at[i] + 2 * (uint32_t)n0));
    };
    // scales and zero points of 128 rows and the tile's eight units of 32 columns: thread's entries 256 i + threadIdx.x,
    // entry = unit * 128 + row
    uint32_t metas[METAS];
    const auto fetch_meta = [&](int t) {
        const int n0 = (b0 + t) * kI4BackN, rows = t < steps ? min(kI4BackN, a.n - n0) : 0;
        const rsrc_t mr = make_rsrc(a.meta + (int64_t)n0 * a.groups, (uint32_t)(rows * a.groups * 4));
#pragma unroll
        for (int i = 0; i < METAS; ++i) {
            const int e = 256 * i + threadIdx.x, row = e & 127, unit = e >> 7;
            const uint32_t g = min(group_at(a, k0 / 32 + unit), (uint32_t)a.groups - 1);
            metas[i] = __builtin_amdgcn_raw_buffer_load_b32(mr, (int)off_if(row < rows, (row * (uint32_t)a.groups + g) * 4), 0, 0);
        }
    };
    const auto keep_meta = [&](int t) {
        meta_t* const table = (meta_t*)(smem + (t & 1) * STAGE + XBYTES);
#pragma unroll
        for (int i = 0; i < METAS; ++i) {
            const int e = 256 * i + threadIdx.x;
            const float s = scale_of(metas[i], a.scale_dtype), z = zero_of(metas[i]);
            table[e] = (meta_t)s;
            table[TABLE + e] = (meta_t)(DT == DK_FP16 ? -1024.0f - z : (-16.0f - z) * s);
        }
    };
    // dwords of the eight rows of a lane in step s (32 rows) of block t
    struct Rows {
        uint32_t d[8];
    };
    const bool cols = k0 + wk < a.kpad;
    const uint32_t w_at = (uint32_t)((k0 + wk) / 2) + 4 * r;
    const auto fetch_w = [&](Rows& f, int t, int s) {
        const int n0 = (b0 + t) * kI4BackN, rows = t < steps && cols ? min(kI4BackN, a.n - n0) : 0;
        const rsrc_t wr = make_rsrc(a.w + (int64_t)n0 * a.ldw, (uint32_t)(rows * a.ldw));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = 32 * s + 8 * q + i;
            f.d[i] = __builtin_amdgcn_raw_buffer_load_b32(wr, (int)off_if(row < rows, row * (uint32_t)a.ldw + w_at), 0, 0);
        }
    };

    float4_t acc[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[c][j] = float4_t{};

    const auto step = [&](const Rows& f, int t, int s) {
        const uint8_t* const stage = smem + (t & 1) * STAGE;
        const meta_t* const table = (const meta_t*)(stage + XBYTES) + ((wk / 32) + (r & 3)) * kI4BackN + 32 * s + 8 * q;
        BackMeta<DT> m;
        m.scale = *(const decltype(m.scale)*)table;
        m.zero = *(const decltype(m.zero)*)(table + TABLE);
        vec x[C];
#pragma unroll
        for (int c = 0; c < C; ++c) x[c] = *(const vec*)(stage + (wm + 16 * c + r) * 256 + 16 * ((4 * s + q) ^ r));
        uint32_t w[4][8];
#pragma unroll
        for (int p = 0; p < 4; ++p) weights_of_pair<DT>(f.d[2 * p], f.d[2 * p + 1], m, p, w[p]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const vec b = __builtin_bit_cast(vec, u32x4_t{w[0][j], w[1][j], w[2][j], w[3][j]});
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c][j] = I4<DT>::mfma(x[c], b, acc[c][j]);
        }
    };

    Rows f[2];
    fetch_meta(0);
    fetch_w(f[0], 0, 0);
    fetch_x(0);
    keep_meta(0);
    fetch_meta(1);
    for (int t = 0; t < steps; ++t) {
        wait_vmcnt<0>();
        lds_barrier();  // stage t is whole, and every wave has read the one before it
        keep_meta(t + 1);
        fetch_w(f[1], t, 1);
        fetch_x(t + 1);
        fetch_meta(t + 2);
        step(f[0], t, 0);
        fetch_w(f[0], t, 2);
        step(f[1], t, 1);
        fetch_w(f[1], t, 3);
        step(f[0], t, 2);
        fetch_w(f[0], t + 1, 0);
        step(f[1], t, 3);
    }
    wait_vmcnt<0>();

    // lane: tokens wm + 16 c + 4 q + e, columns 32 (r & 3) + 8 (r >> 2) + 0 .. 7 of the wave's 128
    const int k = k0 + wk + 32 * (r & 3) + 8 * (r >> 2), left = a.k - k;
    if (left <= 0) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + wm + 16 * c + 4 * q + e;
            if (m >= a.m) continue;
            float8_t v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = acc[c][j][e];
            const int dt = a.splits > 1 ? DK_FP32 : a.y_dtype;
            const int64_t at = a.splits > 1 ? split * a.slab + (int64_t)m * a.k + k : (int64_t)m * a.ldy + k;
            void* const out = a.splits > 1 ? (void*)a.partials : a.y;
            if (dt == DK_FP32) {
                if (left >= 8) store8<DK_FP32>((float*)out + at, v);
                else
                    for (int j = 0; j < 8; ++j)
                        if (j < left) ((float*)out)[at + j] = v[j];
            } else {
                typedef typename Elem<DT>::type E;
                if (left >= 8) store8<DT>((E*)out + at, v);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) store1<DT>((E*)out + at + j, v[j]);
            }
        }
}

// ---- joins and copies ----------------------------------------------------------------------------

// y = sum of the splits' partial sums (in their order) + bias
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Args a, int cols) {
    const int64_t total = (int64_t)a.m * cols, step = (int64_t)gridDim.x * 256 * 4;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += step) {
        typedef float4_t loose4 __attribute__((aligned(4)));
        const int count = (int)min((int64_t)4, total - i);
        float4_t v = {};
        for (int s = 0; s < a.splits; ++s) {
            const float* const p = a.partials + s * a.slab + i;
            if (count == 4) {
                v = v + *(const loose4*)p;
            } else {
                for (int e = 0; e < count; ++e) v[e] += p[e];
            }
        }
        for (int e = 0; e < count; ++e) {
            const int64_t m = (i + e) / cols, n = i + e - m * cols;
            store_out(a, m * a.ldy + n, a.bias != nullptr ? v[e] + load_any(a.bias, a.bias_dtype, n) : v[e]);
        }
    }
}

// rows of 16-bit values to rows of `ld` (a multiple of eight), zeros past their columns
__global__ __launch_bounds__(256) void int4_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, uint16_t* __restrict__ y,
                                                        int64_t rows, int cols, int ld) {
    const int64_t total = rows * (ld / 8), step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / (ld / 8);
        const int c = (int)(i - row * (ld / 8)) * 8;
        typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
        typedef u16x8_t loose __attribute__((aligned(2)));
        u16x8_t v = {};
        const uint16_t* const p = x + row * ldx + c;
        if (c + 8 <= cols) {
            v = *(const loose*)p;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < cols) v[e] = p[e];
        }
        *(u16x8_t*)(y + row * ld + c) = v;
    }
}

// ---- plans and launches --------------------------------------------------------------------------

Int4Plan int4_plan(int64_t m, int64_t n, int64_t k, bool backward) {
    Int4Plan p{};
    const int64_t blocks = (k + kI4Block - 1) / kI4Block;
    if (!backward && m <= kInt4FewM) {
        p.few = true;
        p.tokens = m <= 16 ? 16 : m <= 32 ? 32 : 64;
        const int64_t groups = (n + 15) / 16;
        p.waves = groups < 512 && blocks >= 32 ? 16 : groups < 1024 && blocks >= 16 ? 8 : 4;
        if (p.tokens == 64 && p.waves == 16) p.waves = 8;
        p.splits = 1;
        p.m_tiles = 1;
        p.n_tiles = (int)groups;
        return p;
    }
    const int64_t steps = backward ? (n + kI4BackN - 1) / kI4BackN : blocks;
    p.tokens = backward ? (m <= 32 ? 32 : m <= 64 ? 64 : 128) : kI4TileM;
    p.m_tiles = (int)((m + p.tokens - 1) / p.tokens);
    const int64_t cols = backward ? k : n;
    p.n_tiles = (int)((cols + 255) / 256);
    // splits of the sum until the tiles fill the CUs (the backward's work-groups run two a CU), at least four steps each
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles, fill = backward ? 512 : 256;
    int64_t want = tiles >= fill * 3 / 4 ? 1 : fill / tiles;
    if (want > steps / 4) want = steps / 4;
    if (want < 1) want = 1;
    p.steps_per_split = (int)((steps + want - 1) / want);
    p.splits = (int)((steps + p.steps_per_split - 1) / p.steps_per_split);
    p.partial_bytes = p.splits > 1 ? (int64_t)p.splits * m * cols * 4 : 0;
    return p;
}

template <int DT, int C, int GJ, int P>
static hipError_t launch_few(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    const dim3 grid(p.n_tiles, (a.m + 16 * C - 1) / (16 * C));
    switch (p.waves) {
        case 16:
            if constexpr (C < 4) hipLaunchKernelGGL((int4_few_kernel<DT, C, GJ, 16, P>), grid, dim3(1024), 0, s, a);
            break;
        case 8: hipLaunchKernelGGL((int4_few_kernel<DT, C, GJ, 8, P>), grid, dim3(512), 0, s, a); break;
        default: hipLaunchKernelGGL((int4_few_kernel<DT, C, GJ, 4, P>), grid, dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

template <int DT, int GJ>
static hipError_t launch_forward(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    if (p.few) {
        if (p.tokens == 16) return launch_few<DT, 1, GJ, 4>(a, p, s);
        if (p.tokens == 32) return launch_few<DT, 2, GJ, 2>(a, p, s);
        return launch_few<DT, 4, GJ, 2>(a, p, s);
    }
    constexpr size_t lds = kI4Waves * 64 * 72 * 2 > 2 * kI4StageBytes ? kI4Waves * 64 * 72 * 2 : 2 * kI4StageBytes;
    if (hipError_t e = allow_dynamic_lds((const void*)int4_tile_kernel<DT, GJ>, lds)) return e;
    hipLaunchKernelGGL((int4_tile_kernel<DT, GJ>), dim3(p.m_tiles * p.n_tiles * p.splits), dim3(64 * kI4Waves), lds, s, a);
    return hipGetLastError();
}

template <int DT, int C>
static hipError_t launch_back(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    constexpr size_t lds = int4_back_lds<DT, C>();
    if (hipError_t e = allow_dynamic_lds((const void*)int4_back_kernel<DT, C>, lds)) return e;
    hipLaunchKernelGGL((int4_back_kernel<DT, C>), dim3(p.m_tiles * p.n_tiles * p.splits), dim3(256), lds, s, a);
    return hipGetLastError();
}

template <int DT>
static hipError_t launch_typed(const Int4Args& a, const Int4Plan& p, bool backward, hipStream_t s) {
    if (backward) {
        if (p.tokens == 32) return launch_back<DT, 1>(a, p, s);
        if (p.tokens == 64) return launch_back<DT, 2>(a, p, s);
        return launch_back<DT, 4>(a, p, s);
    }
    if (a.group_units % 4 == 0) return launch_forward<DT, 4>(a, p, s);
    if (a.group_units % 2 == 0) return launch_forward<DT, 2>(a, p, s);
    return launch_forward<DT, 1>(a, p, s);
}

hipError_t launch_int4(Int4Args a, const Int4Plan& p, int dtype, bool backward, hipStream_t s) {
    const int cols = backward ? a.k : a.n, sum = backward ? a.n : a.k;
    a.group_mul = (uint32_t)((0x100000000ull + a.group_units - 1) / (uint64_t)a.group_units);
    a.kpad = (a.k + kI4Block - 1) / kI4Block * kI4Block;
    a.blocks = (sum + 127) / 128;
    a.x_cols = (sum + 7) / 8 * 8;
    a.blocks_per_split = p.steps_per_split;
    a.splits = p.splits;
    a.m_tiles = p.m_tiles;
    a.n_tiles = p.n_tiles;
    a.slab = (int64_t)a.m * cols;
    if (a.padded != nullptr) {
        const int ld = a.x_cols;
        const int64_t items = (int64_t)a.m * (ld / 8), grid = (items + 255) / 256;
        hipLaunchKernelGGL(int4_rows_kernel, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, s, (const uint16_t*)a.x,
                           a.ldx, a.padded, (int64_t)a.m, sum, ld);
        a.x = a.padded;
        a.ldx = ld;
        if (hipError_t e = hipGetLastError()) return e;
    }
    hipError_t e = dtype == DK_FP16 ? launch_typed<DK_FP16>(a, p, backward, s) : launch_typed<DK_BF16>(a, p, backward, s);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t grid = ((int64_t)a.m * cols + 1023) / 1024;
    hipLaunchKernelGGL(int4_join_kernel, dim3((unsigned)(grid < 8192 ? grid : 8192)), dim3(256), 0, s, a, cols);
    return hipGetLastError();
}

}  // namespace dk
