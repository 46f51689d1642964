// Linear layers whose weight holds 4-bit integers with a scale and a zero point for every group of columns of a row:
//   W[n, k] = (code[n, k] - zero[n, k / group]) scale[n, k / group]
//   forward   y[m, n]  = sum over groups g of scale[n, g] (sum over k in g of x[m, k] (code[n, k] - zero[n, g])) + bias[n]
//   backward  dx[m, k] = sum over n of dy[m, n] W[n, k]
// on 16x16x32 MFMAs of the activations' type with fp32 sums. Few tokens: the matrix operands are exact, code - zero a
// small integer, and the scale is applied to a group's fp32 sum: nothing is rounded but the sums and the output. Tiles, and
// the backward, whose sum goes over rows that each have a scale of their own: W is rounded once to 16 bits, as the
// matrix cores take it (at most half a step of the type a weight, which is what a product with a 16-bit weight has).
// Against 64 bits at 4096 tokens of [18944] x 3584, bf16: 0.0022 of the outputs' size, of which 0.0017 their own rounding.
//
// Layout: tiles of 16 rows by 128 columns in 1024 bytes, a row of tiles after the other, so that a wave's load is one
// piece of memory and a lane's 16 bytes are its operands of four MFMAs as they lie: the 16 bytes 16 q + r hold row r,
// their dword j columns 32 j + 8 q + 0 .. 7, column 2 i of those in bits 4 i, column 2 i + 1 in bits 16 + 4 i (a
// shift and a mask leave a pair in the halves of a register). In each MFMA lane l = 16 q + r holds k = 8 q + 0 .. 7 of
// row r of its operand. `meta` holds groups' words, a scale (low 16 bits) and a zero point (next byte), by tile rows, groups
// and the tile's 16 rows.
// From pairs to operands: 0x6400 | q is 1024 + q as fp16, 0x6400 | 16 q is 1024 + 16 q. fp16: one packed subtraction or
// multiply-add leaves q - zero, exactly, one packed product the weight. bf16, and fp16 with bf16 scales (rounded to fp16 before
// the product, a scale below 2^-17 would be off by up to fifteen half steps in a weight, one past 65504 no number): mixed
// multiply-adds give (1024 + q) scale - (1024 + zero) scale in fp32, and one conversion a pair rounds: a scale has 11 bits at
// most and is below 2^117, so both products are exact and the difference is scale (q - zero) without any error (with 1 for the
// scale, q - zero). us, fp16 with fp16 and with bf16 scales: 4096 tokens of [18944] x 3584 forward 460 and 480, backward 485
// and 530.
#include <cstdio>
#include <cstdlib>

#include "elem.h"
#include "gemm_common.h"

namespace dk {

constexpr int kI4Block = 128, kI4Tile = 1024;  // columns of a tile, its bytes

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

// (v & mask) | bits in one instruction: it takes no literals and one scalar register, so the mask is held in one of those
// and the bits in a vector register
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
    asm("" : "+s"(mask));
    asm("" : "+v"(bits));
    return (v & mask) | bits;
}

__device__ __forceinline__ float zero_of(uint32_t meta) { return (float)((meta >> 16) & 0xFF); }

// scale of either 16-bit type
__device__ __forceinline__ float scale_of(uint32_t meta, int scale_dtype) {
    return scale_dtype == DK_BF16 ? I4<DK_BF16>::scale(meta) : I4<DK_FP16>::scale(meta);
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// Which weights are formed in fp32 and rounded at the end: bf16 ones, and fp16 ones with bf16 scales.
constexpr bool i4_wide(int dt, int scale_dtype) { return dt == DK_BF16 || scale_dtype == DK_BF16; }

// two weights as operands of type DT
template <int DT>
__device__ __forceinline__ uint32_t narrow(float a, float b) {
    if constexpr (DT == DK_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, bf16x2_t));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, half2_t));
}

// Constants of a row's group, and operands of a word's columns 0 .. 7: the integers code - zero, or the weights.
template <int DT, bool WIDE = i4_wide(DT, DT)>
struct I4Group;
template <>
struct I4Group<DK_FP16, false> {
    half2_t whole, part, scale;  // -(1024 + zero), -(64 + zero)
    __device__ __forceinline__ void set_zero(uint32_t meta) {
        const _Float16 z = (_Float16)zero_of(meta);
        const _Float16 a = (_Float16)-1024.0f - z, b = (_Float16)-64.0f - z;
        whole = half2_t{a, a};
        part = half2_t{b, b};
    }
    __device__ __forceinline__ void set(uint32_t meta, int) {
        set_zero(meta);
        const _Float16 s = __builtin_bit_cast(_Float16, (uint16_t)meta);
        scale = half2_t{s, s};
    }
    __device__ __forceinline__ half2_t even(uint32_t v) const {
        return __builtin_bit_cast(half2_t, and_or(v, 0x000F000Fu, 0x64006400u)) + whole;
    }
    __device__ __forceinline__ half2_t odd(uint32_t v) const {
        const half2_t sixteenth = half2_t{(_Float16)0.0625f, (_Float16)0.0625f};
        return __builtin_elementwise_fma(__builtin_bit_cast(half2_t, and_or(v, 0x00F000F0u, 0x64006400u)), sixteenth, part);
    }
    static __device__ __forceinline__ half8_t join(half2_t a, half2_t b, half2_t c, half2_t d) {
        return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    __device__ __forceinline__ half8_t integers(uint32_t d) const { return join(even(d), odd(d), even(d >> 8), odd(d >> 8)); }
    __device__ __forceinline__ half8_t weights(uint32_t d) const {
        return join(even(d) * scale, odd(d) * scale, even(d >> 8) * scale, odd(d >> 8) * scale);
    }
};
template <int DT>
struct I4Group<DT, true> {
    typedef typename I4<DT>::vec vec;
    float whole, whole_zero, part, part_zero;  // of 1024 + code, and of 1024 + 16 code
    __device__ __forceinline__ void set_scale(uint32_t meta, float s) {
        const float z = zero_of(meta);
        whole = s;
        whole_zero = (-1024.0f - z) * s;
        part = s * 0.0625f;
        part_zero = (-64.0f - z) * s;
    }
    __device__ __forceinline__ void set_zero(uint32_t meta) {
        float one = 1.0f;
        asm("" : "+v"(one));  // a factor: a product by 1 is made a conversion and a sum
        set_scale(meta, one);
    }
    __device__ __forceinline__ void set(uint32_t meta, int scale_dtype) {
        set_scale(meta, scale_of(meta, DT == DK_FP16 ? DK_BF16 : scale_dtype));
    }
    static __device__ __forceinline__ uint32_t pair(uint32_t v, float by, float plus) {
        const half2_t h = __builtin_bit_cast(half2_t, v);
        return narrow<DT>(__builtin_fmaf((float)h[0], by, plus), __builtin_fmaf((float)h[1], by, plus));
    }
    __device__ __forceinline__ vec weights(uint32_t d) const {
        const uint32_t h = d >> 8;
        return __builtin_bit_cast(vec, u32x4_t{pair(and_or(d, 0x000F000Fu, 0x64006400u), whole, whole_zero),
                                               pair(and_or(d, 0x00F000F0u, 0x64006400u), part, part_zero),
                                               pair(and_or(h, 0x000F000Fu, 0x64006400u), whole, whole_zero),
                                               pair(and_or(h, 0x00F000F0u, 0x64006400u), part, part_zero)});
    }
    __device__ __forceinline__ vec integers(uint32_t d) const { return weights(d); }  // (of set_zero)
};

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
// Bound: the weight's bytes and the latency of a launch's phases. [18944] x 3584 from memory, fp16: 1 token 10.9 us (34 MB and
// 1.2 MB of groups' words, 3.3 TB/s; the first kernel 19), 16 tokens 14.9, 32 tokens 22. [3584] x 18944: 1 to 4 tokens
// 11.6 (bf16 13.8: its unpacking, 32 vector instructions an MFMA); 8, 12 and 16 tokens in two, three and four splits 14.7 (16.7)
// all three, as each of some 224 work-groups has 150 KB of tokens to bring to LDS before its first product, and 3.9 for the join,
// a launch and two round trips (first 31 in all).
// Tokens by 16 (blockIdx.z). The NW waves of a work-group are NW / a.shares tiles of 16 rows by a.shares shares of the split's
// columns, whose sums meet in LDS; each streams its share of the weight to registers, P blocks ahead. The tokens' columns
// of the split are kept in LDS: from the caches with each block they cost the address unit four loads for the
// weight's one, and the L2 as much traffic as the weight from four tokens on ([3584, 18944] at 16 tokens: 22 us that
// way). GJ: the 32-column units a scale is constant over (4, 2 or 1).
typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
typedef u16x8_t u16x8_loose_t __attribute__((aligned(2)));
constexpr int kI4RowPad = 64;  // bytes behind a token's row in LDS: neighbouring rows start in other banks

// (whole loads of a wave)
__host__ __device__ constexpr int few_x_bytes(int m, int blocks) { return (m * (blocks * 256 + kI4RowPad) + 1023) / 1024 * 1024; }

template <int DT, int GJ, int NW, int P>
__global__ __launch_bounds__(64 * NW) void int4_few_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    constexpr int UNITS = 4 / GJ;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int tiles = NW / a.shares, share = wave % a.shares, tile = blockIdx.x * tiles + wave / a.shares;
    const int first = blockIdx.y * a.blocks_per_split, blocks = min(a.blocks_per_split, a.blocks - first);
    const int per = (blocks + a.shares - 1) / a.shares, b0 = share * per;  // blocks of the split
    const int b1 = wave / a.shares < tiles && tile < a.n_tiles ? min(blocks, b0 + per) : 0;

    const int m0 = 16 * blockIdx.z, toks = min(16, a.m - m0);
    const rsrc_t wr = make_rsrc(a.w + ((int64_t)tile * a.kblocks + first) * kI4Tile, (uint32_t)(blocks * kI4Tile));
    const rsrc_t mr = make_rsrc(a.meta + (int64_t)tile * a.groups * 16, (uint32_t)(a.groups * 64));
    struct Stage {
        u32x4_t w;
        uint32_t meta[UNITS];
    };
    Stage st[P];
    const auto fetch = [&](Stage& s, int b) {
        const bool live = b < b1;
        s.w = bload128(wr, off_if(live, kI4Tile * (uint32_t)b + 16 * lane));
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            // (a last block's units past k have no group: they read the last one's, for x of zeros)
            const uint32_t g = min(group_at(a, 4 * (first + b) + GJ * u), (uint32_t)a.groups - 1);
            s.meta[u] = __builtin_amdgcn_raw_buffer_load_b32(mr, (int)off_if(live, 64 * g + 4 * r), 0, 0);
        }
    };
    // the tokens' rows, zeros behind their columns
    const int pitch = blocks * 256 + kI4RowPad;
    {
        const uint16_t* const x = (const uint16_t*)a.x + m0 * a.ldx;
        const int chunks = pitch / 16, total = toks * chunks, c0 = first * kI4Block;
        if (!a.loose) {
            const rsrc_t xr = make_rsrc(x, (uint32_t)(((toks - 1) * a.ldx + a.k) * 2));
            for (int i = 64 * wave; i < total; i += 64 * NW) {
                const int row = (i + lane) / chunks, c = c0 + 8 * (i + lane - row * chunks);
                bload128_lds(xr, smem + 16 * i,
                             off_if(row < toks && c < min(a.k, c0 + blocks * kI4Block), (uint32_t)(row * a.ldx + c) * 2));
            }
        } else {
            // rows that start anywhere, or end inside eight columns
            for (int i = threadIdx.x; i < total; i += 64 * NW) {
                const int row = i / chunks, c = c0 + 8 * (i - row * chunks), left = min(a.k, c0 + blocks * kI4Block) - c;
                u16x8_t v = {};
                const uint16_t* const p = x + row * a.ldx + c;
                if (left >= 8) {
                    v = *(const u16x8_loose_t*)p;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < left) v[e] = p[e];
                }
                *(u16x8_t*)(smem + 16 * i) = v;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) fetch(st[p], b0 + p);
    wait_vmcnt<P>();  // the tokens, and of the weight (and its scales) some
    lds_barrier();
    const uint8_t* const x_row = smem + (r < toks ? r : 0) * pitch + 16 * q;  // (other rows' results are not stored)

    float4_t acc = {};
    const auto compute = [&](const Stage& s, int b) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t meta = s.meta[u];
            I4Group<DT> group;
            group.set_zero(meta);
            float4_t t = {};
#pragma unroll
            for (int j = GJ * u; j < GJ * (u + 1); ++j) {
                const vec w = group.integers(s.w[j]), x = *(const vec*)(x_row + 256 * b + 64 * j);
                t = I4<DT>::mfma(x, w, t);
            }
            const float scale = scale_of(meta, a.scale_dtype);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(t[i], scale, acc[i]);
        }
    };
    int b = b0;
    for (; b + P < b1; b += P) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            compute(st[p], b + p);
            fetch(st[p], b + p + P);
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
        if (b + p < b1) compute(st[p], b + p);

    // lane: row 16 tile + r, tokens 4 q + i
    __syncthreads();
    float(*const sums)[4][64] = (float(*)[4][64])smem;
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < tiles * 256; e += 64 * NW) {
        const int t = e >> 8, l = e & 63, m = m0 + 4 * (l >> 4) + ((e >> 6) & 3), n = 16 * (blockIdx.x * tiles + t) + (l & 15);
        if (m >= a.m || n >= a.n) continue;
        float v = 0.0f;
        for (int w = 0; w < a.shares; ++w) v += sums[t * a.shares + w][(e >> 6) & 3][l];
        if (a.splits > 1) {
            a.partials[blockIdx.y * a.slab + (int64_t)m * a.n + n] = v;
        } else {
            if (a.bias != nullptr) v += load_any(a.bias, a.bias_dtype, n);
            store_out(a, (int64_t)m * a.ldy + n, v);
        }
    }
}

// ---- tiles ---------------------------------------------------------------------------------------
// Bound: the matrix cores' and vector units' cycles and the loads' issue between them. 4096 tokens of [18944] x 3584, bf16:
// forward 470 to 510 us (1.1 to 1.18 PFLOP/s, matrix cores busy 51% of all cycles; the first kernel 1479), backward 540 to
// 595 (1.0 PFLOP/s, 42%; first 1364), where a library product of the same sizes with a 16-bit weight takes 537 to 547. 830
// tokens of [8960] x 1536, fp16: forward 27 to 31 us (245 work-groups of 12 blocks; such a library product 29), backward 40
// with the join of six splits (45), 40 + 7 from memory. Waves of 64 by 64 in the smaller tiles, as in the largest, unpack
// each weight twice: 34 and 43.5 us.
// Tiles of 32 C tokens by 256 rows of the weight (forward) or 256 columns (backward), eight waves: with 256 tokens of 128 by
// 64, with fewer of all tokens by 32, so that no weight is unpacked twice (kI4Across: waves along the tokens). The sum
// goes in steps of 64 terms through a ring of three stages of LDS, filled by loads that go there directly: one wait and
// one barrier a step, loads two steps ahead. The weight stays in 4 bits up to each wave's registers.
// W is rounded to the activations' type here, once.
constexpr int kI4Waves = 8, kI4TileN = 256, kI4Step = 64, kI4Ring = 3;
template <int C>
constexpr int kI4Across = C == 8 ? 2 : 1;

// An offset in a stage that every step adds its stage's to: held as it is, or each read's would be formed again.
__device__ __forceinline__ uint32_t held(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// 16-byte chunk of a row of 128 bytes: neighbouring rows share the banks' two halves, pairs of rows are permuted
__device__ __forceinline__ int chunk_key(int row) { return (row >> 1) & 7; }

// Consecutive tiles on one XCD, token tiles fastest within bands of eight, so that the tiles of an XCD at one time share
// rows of both operands.
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

// The activations' part of a stage: rows of 64 terms (128 bytes), and a wave's loads of a step. Steps are fetched in
// turn: `src` starts at the next one's columns, of which `left` are there (none behind the last).
template <int C>
struct I4Tokens {
    static constexpr int TM = 32 * C, BYTES = TM * 128, LOADS = BYTES / 1024 / kI4Waves;
    const uint16_t* from;
    uint32_t bytes;
    int left, wave;
    uint32_t at[LOADS];
    int col[LOADS];
    __device__ __forceinline__ void set(const Int4Args& a, int m0, int c0, int cols, int w, int lane) {
        const int toks = min(TM, a.m - m0);
        wave = w;
        from = (const uint16_t*)a.x + (int64_t)m0 * a.ldx + c0;
        left = min(cols, a.x_cols - c0);
        bytes = (uint32_t)(((toks - 1) * a.ldx + left) * 2);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = 8 * (wave * LOADS + i) + (lane >> 3);
            col[i] = 8 * ((lane & 7) ^ chunk_key(row));
            at[i] = off_if(row < toks, (row * (uint32_t)a.ldx + col[i]) * 2);
        }
    }
    __device__ __forceinline__ void load(uint8_t* stage, int i) const {
        bload128_lds(make_rsrc(from, left > 0 ? bytes : 0), stage + 1024 * (wave * LOADS + i), off_if(col[i] < left, at[i]));
    }
    __device__ __forceinline__ void turn() {
        from += kI4Step;
        bytes -= 2 * kI4Step;
        left -= kI4Step;
    }
    __device__ __forceinline__ void fetch(uint8_t* stage) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load(stage, i);
        turn();
    }
};

// N neighbouring outputs, of which `left` are there
template <int DT, int N>
__device__ __forceinline__ void put(void* y, int64_t at, float __attribute__((ext_vector_type(N))) v, int left) {
    typedef typename Elem<DT>::type E;
    typedef E vec_n __attribute__((ext_vector_type(N)));
    typedef vec_n loose_n __attribute__((aligned(sizeof(E))));
    asm("" : "+v"(v));
    if (left >= N) {
        *(loose_n*)((E*)y + at) = __builtin_convertvector(v, vec_n);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < left) ((E*)y)[at + e] = (E)v[e];
    }
}

// ---- forward, many tokens: two steps a block of 128 columns; the weight's block and its groups' words every other step
constexpr int kI4WBytes = kI4TileN * 64;
template <int C, int GJ>
constexpr size_t int4_tile_lds() {
    constexpr size_t ring = kI4Ring * (I4Tokens<C>::BYTES + kI4WBytes + 4 / GJ * kI4TileN * 4);
    constexpr size_t out = kI4Waves * 64 * (32 * kI4Across<C> + 8) * 2;
    return ring > out ? ring : out;
}

template <int DT, bool WIDE, int C, int GJ>
__global__ __launch_bounds__(64 * kI4Waves, 2) void int4_tile_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    // a wave: F times 16 tokens by R times 16 rows
    constexpr int WM = kI4Across<C>, F = 2 * C / WM, R = 2 * WM;
    constexpr int UNITS = 4 / GJ, XB = I4Tokens<C>::BYTES, WB = kI4WBytes + UNITS * kI4TileN * 4;
    constexpr int METAS = UNITS == 4 ? 2 : 1, WLOADS = 2 + METAS;  // a wave's loads of a block
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    int mt, nt, split;
    tile_of(a, mt, nt, split);
    const int m0 = mt * 32 * C, n0 = nt * kI4TileN;
    const int wm = wave % WM * 16 * F, wn = wave / WM * 16 * R;
    const int b0 = split * a.blocks_per_split, blocks = min(a.blocks_per_split, a.blocks - b0);

    I4Tokens<C> x;
    x.set(a, m0, b0 * kI4Block, blocks * kI4Block, wave, lane);
    const int tiles = (min(kI4TileN, a.n - n0) + 15) / 16;
    const rsrc_t wr = make_rsrc(a.w + (int64_t)(n0 / 16) * a.kblocks * kI4Tile, (uint32_t)(tiles * a.kblocks * kI4Tile));
    const rsrc_t mr = make_rsrc(a.meta + (int64_t)n0 * a.groups, (uint32_t)(tiles * a.groups * 64));
    uint8_t* const weights = smem + kI4Ring * XB;
    const auto fetch_x = [&](int h) { x.fetch(smem + (h % kI4Ring) * XB); };
    const auto fetch_w = [&](int b) {
        uint8_t* const stage = weights + (b % kI4Ring) * WB;
        const bool live = b < blocks;
#pragma unroll
        for (int i = 0; i < 2; ++i)  // a tile a load
            bload128_lds(wr, stage + kI4Tile * (2 * wave + i),
                         off_if(live, kI4Tile * ((2 * wave + i) * (uint32_t)a.kblocks + (uint32_t)(b0 + b)) + 16 * lane));
#pragma unroll
        for (int i = 0; i < METAS; ++i) {  // 64 rows of one unit a load; with one unit waves 4 to 7 repeat 0 to 3's
            const int load = UNITS == 1 ? wave & 3 : METAS * wave + i, u = load >> 2;
            const uint32_t tile = 4 * (load & 3) + q;
            const uint32_t g = min(group_at(a, 4 * (b0 + b) + GJ * u), (uint32_t)a.groups - 1);
            bload32_lds(mr, stage + kI4WBytes + 256 * load, off_if(live, 64 * (tile * (uint32_t)a.groups + g) + 4 * r));
        }
    };

    float4_t acc[R][F];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < F; ++c) acc[i][c] = float4_t{};

    // A step is four parts: each 32 terms by half of the tokens. Operands of a part are read in the one before, across
    // the steps too: the wait and the barrier of a step come before its last part, when all of it has been read.
    constexpr int H = F / 2;
    vec xv[2][H], wv[2][R];
    u32x4_t raw[R];
    I4Group<DT, WIDE> group[R];
    const uint32_t x_off[2] = {held((wm + r) * 128 + 16 * (q ^ chunk_key(r))), held((wm + r) * 128 + 16 * ((4 + q) ^ chunk_key(r)))};
    const uint32_t w_off = held(kI4Ring * XB + wn * 64 + 16 * lane);
    const uint32_t g_off = held(kI4Ring * XB + kI4WBytes + 4 * (wn + r));
    // xs, ws: where the step's tokens and the block's weights are
    const auto read_x = [&](uint32_t xs, int part) {
        const uint8_t* const at = smem + (x_off[part >> 1] + xs);
#pragma unroll
        for (int c = 0; c < H; ++c) xv[part & 1][c] = *(const vec*)(at + (H * (part & 1) + c) * 2048);
    };
    const auto read_raw = [&](uint32_t ws) {
        const uint8_t* const at = smem + (w_off + ws);
#pragma unroll
        for (int i = 0; i < R; ++i) raw[i] = *(const u32x4_t*)(at + kI4Tile * i);
    };
    // operands of slice j (32 columns) of a block
    const auto unpack = [&](uint32_t ws, int j) {
        const uint8_t* const at = smem + (g_off + ws);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (j % GJ == 0) {
                group[i].set(*(const uint32_t*)(at + 4 * (kI4TileN * (j / GJ) + 16 * i)), a.scale_dtype);
                // (else fp16's rows are set at once, early, and 256 tokens spill)
                if constexpr (DT == DK_FP16) __builtin_amdgcn_sched_barrier(0);
            }
            wv[j & 1][i] = group[i].weights(raw[i][j]);
        }
    };
    const auto multiply = [&](int v) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < H; ++c) {
                float4_t& s = acc[i][H * (v & 1) + c];
                s = I4<DT>::mfma(xv[v & 1][c], wv[(v >> 1) & 1][i], s);
            }
    };
    constexpr int GROUP = I4Tokens<C>::LOADS + WLOADS;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        fetch_x(i);
        if (i < 2) fetch_w(i);
    }
    wait_vmcnt<2 * GROUP - WLOADS>();
    lds_barrier();
    uint32_t xs = 0, ws = 0, next_ws = 0;
    read_raw(0);
    read_x(0, 0);
    unpack(0, 0);
    for (int b = 0; b < blocks; ++b) {
#pragma unroll
        for (int v = 0; v < 8; ++v) {  // parts of two steps
            if ((v & 3) == 3) {
                wait_vmcnt<GROUP>();  // all but the newest step's and the newest block's
                lds_barrier();
                fetch_x(2 * b + (v >> 2) + 3);
                xs = xs == 2 * XB ? 0 : xs + XB;
                read_x(xs, 0);
            } else {
                read_x(xs, (v & 3) + 1);
            }
            if (v == 0) fetch_w(b + 2);  // (its stage is free since the barrier before)
            multiply(v);
            if (v == 7) ws = next_ws;
            if (v & 1) unpack(ws, ((v >> 1) + 1) & 3);
            if (v == 5) {  // (the next block is there since the step before)
                next_ws = ws == 2 * WB ? 0 : ws + WB;
                read_raw(next_ws);
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
            for (int c = 0; c < F; ++c)
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
    // 16-bit outputs leave as pieces of 16 bytes: 64 tokens of the wave's rows at a time through LDS
    constexpr int PART = 4, PITCH = 16 * R + 8, PIECES = 2 * R;  // of a token
    typedef typename Elem<DT>::type E;
    E* const mine = (E*)smem + wave * 16 * PART * PITCH;
#pragma unroll
    for (int part = 0; part < F / PART; ++part) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int n = n0 + wn + 16 * i + r;
            const float bias = a.bias != nullptr && n < a.n ? load_any(a.bias, a.bias_dtype, n) : 0.0f;
#pragma unroll
            for (int c = 0; c < PART; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    store1<DT>(mine + (16 * c + 4 * q + e) * PITCH + 16 * i + r, acc[i][part * PART + c][e] + bias);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < PIECES; ++s) {
            const int row = 64 / PIECES * s + lane / PIECES, piece = 8 * (lane % PIECES);
            const int m = m0 + wm + 16 * PART * part + row, n = n0 + wn + piece;
            if (m >= a.m || n >= a.n) continue;
            const E* const from = mine + row * PITCH + piece;
            E* const to = (E*)a.y + (int64_t)m * a.ldy + n;
            if (n + 8 <= a.n) {
                *(typename Elem<DT>::loose*)to = *(const typename Elem<DT>::vec*)from;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < a.n) to[e] = from[e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- backward ------------------------------------------------------------------------------------
// The weight's layout is the forward's. Lanes of an MFMA operand that share a word hold different columns of it, each of
// its eight rows' words: with 64 columns a wave lanes r and r + 8 four each (as many MFMAs), with 32 lanes 4 q' to 4 q' + 3
// two. The bytes with those columns of two rows' words, joined in one register, unpack to pairs along the rows. Rows' scales and zero points go through tables of 64 rows by the tile's eight units
// of 32 columns: their words come a step before the step's other loads, and the threads (an entry each) make the tables
// of the next step.
constexpr int kI4BackUnits = 8, kI4Entries = kI4BackUnits * kI4Step;
// a unit's rows in a table: padded, so that the two units that a wave reads use different banks
constexpr int kI4Unit = kI4Step + 32, kI4Table = kI4BackUnits * kI4Unit;

template <int DT, bool WIDE>
struct BackRows;  // of the eight rows of a lane
template <>
struct BackRows<DK_FP16, false> {
    typedef _Float16 elem;
    half8_t scale, zero;  // -(1024 + zero)
    static __device__ __forceinline__ void keep(elem* table, int e, uint32_t meta, int) {
        table[e] = __builtin_bit_cast(_Float16, (uint16_t)meta);
        table[kI4Table + e] = (elem)(-1024.0f - zero_of(meta));
    }
    // weights of rows 2 p and 2 p + 1: 1024 + code
    __device__ __forceinline__ uint32_t pair(uint32_t v, int p) const {
        const half2_t w = __builtin_bit_cast(half2_t, v) + half2_t{zero[2 * p], zero[2 * p + 1]};
        return __builtin_bit_cast(uint32_t, w * half2_t{scale[2 * p], scale[2 * p + 1]});
    }
};
template <int DT>
struct BackRows<DT, true> {
    typedef float elem;
    float8_t scale, zero;  // -(1024 + zero) scale
    static __device__ __forceinline__ void keep(elem* table, int e, uint32_t meta, int scale_dtype) {
        const float s = scale_of(meta, DT == DK_FP16 ? DK_BF16 : scale_dtype);
        table[e] = s;
        table[kI4Table + e] = (-1024.0f - zero_of(meta)) * s;
    }
    __device__ __forceinline__ uint32_t pair(uint32_t v, int p) const {
        const half2_t h = __builtin_bit_cast(half2_t, v);
        return narrow<DT>(__builtin_fmaf((float)h[0], scale[2 * p], zero[2 * p]),
                          __builtin_fmaf((float)h[1], scale[2 * p + 1], zero[2 * p + 1]));
    }
};

template <bool WIDE, int C>
constexpr int kI4BackVector = (C == 8 ? (WIDE ? 80 : 72) : (WIDE ? 48 : 40)) / (2 * C);

// Order of a part's instructions: V vector ones behind each of M matrix ones, a load every L of them. Issued at once, the
// loads of eight waves and the arithmetic of their addresses hold up the matrix instructions behind them: 4096 tokens of
// [18944] x 3584, bf16, 641 us that way, 542 spread. (The forward has no registers left for it: ordered so it spills, 570
// us for 485.)
template <int M, int V, int L = 1 << 20>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __builtin_amdgcn_sched_group_barrier(8, 1, 0);
        if (i % L == 0 && L <= M) __builtin_amdgcn_sched_group_barrier(16, 1, 0);
        __builtin_amdgcn_sched_group_barrier(2, V, 0);
    }
}

constexpr int kI4BackWBytes = kI4Step * 128;  // 64 rows of 256 columns
template <int DT, bool WIDE, int C>
constexpr int int4_back_stage() {
    return I4Tokens<C>::BYTES + kI4BackWBytes + 2 * kI4Table * (int)sizeof(typename BackRows<DT, WIDE>::elem);
}

template <int DT, bool WIDE, int C>
__global__ __launch_bounds__(64 * kI4Waves, 2) void int4_back_kernel(const Int4Args a) {
    typedef typename I4<DT>::vec vec;
    typedef typename BackRows<DT, WIDE>::elem meta_t;
    // a wave: F times 16 tokens by J times 16 columns
    constexpr int WM = kI4Across<C>, F = 2 * C / WM, J = 2 * WM;
    constexpr int XB = I4Tokens<C>::BYTES, STAGE = int4_back_stage<DT, WIDE, C>();
    extern __shared__ __attribute__((aligned(32))) uint8_t smem[];
    uint32_t* const raw = (uint32_t*)(smem + kI4Ring * STAGE);  // four steps' words of the groups
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    int mt, kt, split;
    tile_of(a, mt, kt, split);
    const int m0 = mt * 32 * C, k0 = kt * 256;
    const int wm = wave % WM * 16 * F, wk = wave / WM;  // the wave's columns: 16 J wk and on
    const int n_begin = split * a.blocks_per_split * kI4Block;
    const int n_end = min(a.n, n_begin + a.blocks_per_split * kI4Block), steps = (n_end - n_begin + kI4Step - 1) / kI4Step;

    I4Tokens<C> x;
    x.set(a, m0, n_begin, a.blocks_per_split * kI4Block, wave, lane);
    // Words of a stage: row 8 q + i of a step's half lies so that the four rows that a read takes (q = 0 .. 3) use different
    // banks: chunks swap halves of the row by bit 3 of the row, rows swap places in their pair by bit 4.
    const int w_slot = 8 * wave + (lane >> 3), w_row = w_slot ^ ((w_slot >> 4) & 1);
    const int w_chunk = (lane & 7) ^ (((w_row >> 3) & 1) << 2);
    const uint32_t w_block = k0 / kI4Block + (w_chunk >> 2);
    const bool w_live = w_block < (uint32_t)a.kblocks;
    const uint32_t w_at = kI4Tile * ((w_row >> 4) * (uint32_t)a.kblocks + w_block) + 16 * (16 * (w_chunk & 3) + (w_row & 15));
    const uint32_t e_group = min(group_at(a, k0 / 32 + (threadIdx.x >> 6)), (uint32_t)a.groups - 1);
    // steps are fetched in turn: the next one's tiles and words of the groups, and how many rows are left for them
    const uint8_t* w_from = a.w + (int64_t)(n_begin / 16) * a.kblocks * kI4Tile;
    const uint32_t* m_from = a.meta + (int64_t)n_begin * a.groups;
    int w_left = n_end - n_begin, m_left = w_left;
    const uint32_t m_at = 64 * (q * (uint32_t)a.groups + e_group) + 4 * r;
    const auto tiles_of = [](int rows) { return rows <= 0 ? 0 : min(4, (rows + 15) / 16); };
    const auto fetch_w = [&](uint8_t* stage) {
        bload128_lds(make_rsrc(w_from, (uint32_t)(tiles_of(w_left) * a.kblocks * kI4Tile)), stage + XB + 1024 * wave, off_if(w_live, w_at));
        w_from += (int64_t)(4 * kI4Tile) * a.kblocks;
        w_left -= kI4Step;
    };
    const auto fetch_meta = [&](int h) {
        bload32_lds(make_rsrc(m_from, (uint32_t)(tiles_of(m_left) * a.groups * 64)), raw + (h & 3) * kI4Entries + 64 * wave, m_at);
        m_from += (int64_t)kI4Step * a.groups;
        m_left -= kI4Step;
    };
    const auto stage_of = [&](int h) { return smem + (h % kI4Ring) * STAGE; };
    const auto table = [&](int h) { return (meta_t*)(smem + (h % kI4Ring) * STAGE + XB + kI4BackWBytes); };

    float4_t acc[F][J];
#pragma unroll
    for (int c = 0; c < F; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j) acc[c][j] = float4_t{};

    // This lane's word of a row is word `word` of chunk 4 (unit / 4) + qw, its columns 8 qw + own and on of the unit. Its
    // bytes: of each half of two rows' words, the one that holds its columns, of which two begin at bit `low`.
    const int unit = WM == 2 ? 2 * wk + (r & 1) : wk, qw = WM == 2 ? (r >> 1) & 3 : r >> 2, word = unit & 3;
    const int chunk = 4 * (unit >> 2) + qw, own = WM == 2 ? 4 * (r >> 3) : 2 * (r & 3), low = 4 * (r & 1);
    const uint32_t pick = own < 4 ? 0x06040200u : 0x07050301u;
    // the parts of a step as in the forward
    constexpr int H = F / 2;
    vec xv[2][H], wv[2][J];
    uint32_t d[8];
    BackRows<DT, WIDE> rows;
    const uint32_t x_off[2] = {held((wm + r) * 128 + 16 * (q ^ chunk_key(r))), held((wm + r) * 128 + 16 * ((4 + q) ^ chunk_key(r)))};
    // (row 8 q + i lies at 8 q + i ^ bit 4 of it, which is bit 1 of q)
    const uint32_t w_off = XB + 8 * q * 128 + 16 * (chunk ^ ((q & 1) << 2)) + 4 * word, swap = 128 * ((q >> 1) & 1);
    const uint32_t w_even = held(w_off + swap), w_odd = held(w_off - swap);
    const uint32_t t_off = held(XB + kI4BackWBytes + (unit * kI4Unit + 8 * q) * (uint32_t)sizeof(meta_t));
    // at: where the step's stage is
    const auto read_x = [&](uint32_t at, int part) {
        const uint8_t* const p = smem + (x_off[part >> 1] + at);
#pragma unroll
        for (int c = 0; c < H; ++c) xv[part & 1][c] = *(const vec*)(p + (H * (part & 1) + c) * 2048);
    };
    const auto read_w = [&](uint32_t at, int s) {
        const uint8_t *const even = smem + (w_even + at) + 4096 * s, *const odd = smem + (w_odd + at) + 4096 * s;
        const uint8_t* const t = smem + (t_off + at) + 32 * s * sizeof(meta_t);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = *(const uint32_t*)((i & 1 ? odd : even) + 128 * i);
        rows.scale = *(const decltype(rows.scale)*)t;
        rows.zero = *(const decltype(rows.zero)*)(t + kI4Table * sizeof(meta_t));
    };
    const auto unpack = [&](int s) {
        uint32_t w[J][4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            // nibbles of row 2 p: columns 0 2 1 3, then of row 2 p + 1
            uint32_t v = __builtin_amdgcn_perm(d[2 * p + 1], d[2 * p], pick);
            if constexpr (WM == 1) v >>= low;
            w[0][p] = rows.pair(and_or(v, 0x000F000Fu, 0x64006400u), p);
            w[1][p] = rows.pair(and_or(v >> 8, 0x000F000Fu, 0x64006400u), p);
            if constexpr (WM == 2) {
                w[2][p] = rows.pair(and_or(v >> 4, 0x000F000Fu, 0x64006400u), p);
                w[3][p] = rows.pair(and_or(v >> 12, 0x000F000Fu, 0x64006400u), p);
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) wv[s][j] = __builtin_bit_cast(vec, u32x4_t{w[j][0], w[j][1], w[j][2], w[j][3]});
    };
    const auto multiply = [&](int part) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int c = 0; c < H; ++c) {
                float4_t& t = acc[H * (part & 1) + c][j];
                t = I4<DT>::mfma(xv[part & 1][c], wv[part >> 1][j], t);
            }
    };
    const auto keep = [&](int h) {  // (a wave's own words)
        BackRows<DT, WIDE>::keep(table(h), kI4Unit * wave + lane, raw[(h & 3) * kI4Entries + threadIdx.x], a.scale_dtype);
    };
    constexpr int GROUP = I4Tokens<C>::LOADS + 2;
    fetch_meta(0);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        fetch_meta(i + 1);
        x.fetch(stage_of(i));
        fetch_w(stage_of(i));
    }
    wait_vmcnt<2 * GROUP>();
    keep(0);
    lds_barrier();
    uint32_t at = 0;
    read_x(0, 0);
    read_w(0, 0);
    unpack(0);
    for (int h = 0; h < steps; ++h) {
        read_x(at, 1);
        read_w(at, 1);
        multiply(0);
        keep(h + 1);
        __builtin_amdgcn_sched_barrier(0);
        read_x(at, 2);
        multiply(1);
        unpack(1);
        interleave<2 * C, kI4BackVector<WIDE, C>>();
        __builtin_amdgcn_sched_barrier(0);
        read_x(at, 3);
        multiply(2);
        wait_vmcnt<GROUP>();  // all but the newest step's
        lds_barrier();
        at = at == 2 * STAGE ? 0 : at + STAGE;
        read_w(at, 0);
        read_x(at, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(3);
        unpack(0);
        fetch_meta(h + 4);
        x.fetch(stage_of(h + 3));
        fetch_w(stage_of(h + 3));
        interleave<2 * C, kI4BackVector<WIDE, C>, (2 * C > GROUP ? 2 * C / GROUP : 1)>();
        __builtin_amdgcn_sched_barrier(0);
    }
    wait_vmcnt<0>();

    // lane: tokens wm + 16 c + 4 q + e, J columns
    typedef float out_t __attribute__((ext_vector_type(J)));
    const int k = k0 + 32 * unit + 8 * qw + own, left = a.k - k;
    if (left <= 0) return;
#pragma unroll
    for (int c = 0; c < F; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + wm + 16 * c + 4 * q + e;
            if (m >= a.m) continue;
            out_t v;
#pragma unroll
            for (int j = 0; j < J; ++j) v[j] = acc[c][j][e];
            if (a.splits > 1)
                put<DK_FP32, J>(a.partials, split * a.slab + (int64_t)m * a.k + k, v, left);
            else if (a.y_dtype == DK_FP32)
                put<DK_FP32, J>(a.y, (int64_t)m * a.ldy + k, v, left);
            else
                put<DT, J>(a.y, (int64_t)m * a.ldy + k, v, left);
        }
}

// ---- joins and copies ----------------------------------------------------------------------------

// y = sum of the splits' partial sums (in their order) + bias; four columns a thread
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Args a, int cols) {
    typedef float4_t loose4 __attribute__((aligned(4)));
    const int n = 4 * (blockIdx.x * 256 + threadIdx.x), left = cols - n;
    if (left <= 0) return;
    float4_t bias = {};
    if (a.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) bias[e] = load_any(a.bias, a.bias_dtype, n + e);
    }
    for (int64_t m = blockIdx.y; m < a.m; m += gridDim.y) {
        const float* p = a.partials + m * cols + n;
        float4_t v = {};
        if (left >= 4) {
            int s = 0;
            for (; s + 4 <= a.splits; s += 4) {
                float4_t t[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = *(const loose4*)(p + e * a.slab);
#pragma unroll
                for (int e = 0; e < 4; ++e) v = v + t[e];
                p += 4 * a.slab;
            }
            for (; s < a.splits; ++s, p += a.slab) v = v + *(const loose4*)p;
        } else {
            for (int s = 0; s < a.splits; ++s, p += a.slab) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < left) v[e] += p[e];
            }
        }
        v = v + bias;
        const int64_t at = m * a.ldy + n;
        if (a.y_dtype == DK_FP32)
            put<DK_FP32, 4>(a.y, at, v, left);
        else if (a.y_dtype == DK_BF16)
            put<DK_BF16, 4>(a.y, at, v, left);
        else
            put<DK_FP16, 4>(a.y, at, v, left);
    }
}

// rows of 16-bit values to rows of `ld` (a multiple of eight), zeros past their columns
__global__ __launch_bounds__(256) void int4_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, uint16_t* __restrict__ y,
                                                        int64_t rows, int cols, int ld) {
    const int64_t total = rows * (ld / 8), step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / (ld / 8);
        const int c = (int)(i - row * (ld / 8)) * 8;
        u16x8_t v = {};
        const uint16_t* const p = x + row * ldx + c;
        if (c + 8 <= cols) {
            v = *(const u16x8_loose_t*)p;
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
    // Tokens by 16 with the weight streamed to registers for each: up to 32, up to 64 on weights whose tiles are mostly start
    // and end. For both types, although tiles would take bf16 less time past 16 tokens of large weights: streamed, no weight is
    // rounded. us, streamed and by the best tiles, fp16 / bf16: [18944] x 3584 at 32 tokens 19.8 and 20.7 / 26.1 and 21.2,
    // [3584] x 18944 18.6 and 22.1 / 23.1 and 22.4; at 64 [4096] x 4096 9.6 and 16.7 / 11.5 and 17.1, [8960] x 1536 12.2 and
    // 15.3 / 15.2 and 15.5, [5120] x 5120, past the bound, 18.3 and 18.7 / 22.8 and 19.5.
    const bool small = n * ((k + 7) / 8 * 8) <= (int64_t(1) << 24);
    if (!backward && std::getenv("DECIK_INT4_PLAN") == nullptr && m <= (small ? kInt4FewSmallM : kInt4FewM)) {
        p.few = true;
        p.tokens = 16;
        p.m_tiles = (int)((m + 15) / 16);
        const int toks = m < 16 ? (int)m : 16;
        p.n_tiles = (int)((n + 15) / 16);
        // Splits where the tokens' columns do not fit the LDS. Where they take much of it and there are more row tiles than CUs,
        // work-groups of 16 waves with as many tiles as one round of the CUs needs (over all tokens and splits: [4096] x 4096
        // at 48 tokens 16.0 us with three tiles, a round and two work-groups, 9.4 with four); else one tile a work-group, four or eight
        // waves sharing its columns. us, in turn with four waves, eight, sixteen sharing and the choice: [18944] x 3584 at
        // 1 token 11.1, 11.0, 13.6, 11.0; at 16 30.4, 24.7, 26.4, 14.1; [8960] x 1536 at 1 token 4.8, 5.2, 6.9, 4.8; at 16 6.3,
        // 6.7, 8.3, 5.6; [4096] x 4096 at 4 tokens 5.9, 5.3, 5.3, 5.3.
        p.splits = 1;
        while (few_x_bytes(toks, (int)((blocks + p.splits - 1) / p.splits)) > kInt4FewLds) ++p.splits;
        const int x_bytes = few_x_bytes(toks, (int)((blocks + p.splits - 1) / p.splits));
        const int64_t groups = (int64_t)p.n_tiles * p.splits * p.m_tiles;
        if (x_bytes > 32768 && groups > 256) {
            int tiles = 2;
            while (tiles < 16 && (p.n_tiles + tiles - 1) / tiles * (int64_t)(p.splits * p.m_tiles) > 256) ++tiles;
            p.waves = 16;
            p.shares = 16 / tiles;
        } else {
            p.waves = p.shares = p.n_tiles >= 512 && blocks <= 16 ? 4 : 8;
        }
        p.steps_per_split = (int)((blocks + p.splits - 1) / p.splits);
        p.splits = (int)((blocks + p.steps_per_split - 1) / p.steps_per_split);
        p.partial_bytes = p.splits > 1 ? (int64_t)p.splits * m * n * 4 : 0;
        return p;
    }
    // Tokens a tile (256, 128 or 64) and splits of the sum: the least estimate of the time. A round of the CUs takes the times
    // below for a block of 128 terms and for its start and end (tiles of 64 tokens run two work-groups a CU, one alone
    // takes less), a split's partial sums go to memory and back, their join takes a launch. Fitted to 1300 timed plans of 70
    // products (fp16, 64 to 4096 tokens, weights from [512] x 3584 to [18944] x 3584), launches included: estimates are off by 10%
    // forward and 8% backward at the mean, 44% at most ([830, 8960] x 1536 forward 22 us for 29), mostly too low; the
    // chosen plan is off the best one's time by 0.4% at the mean and 5% at most. Measured against the choice: [830, 8960] x 1536
    // forward 29 us (tiles of 64 tokens 33, of 256 45), backward 42 in six splits of 128 (10 of 256: 47, 6 of 64: 48).
    // (Tuning hook, read on every call: DECIK_INT4_PLAN = "tokens,splits" forces a plan.)
    const int64_t cols = backward ? k : n, steps = backward ? (n + kI4Block - 1) / kI4Block : blocks;
    const int most = (backward ? n : k) < kInt4LongRow ? 256 : 64;
    p.n_tiles = (int)((cols + kI4TileN - 1) / kI4TileN);
    int forced_tokens = 0, forced_splits = 0;
    if (const char* v = std::getenv("DECIK_INT4_PLAN"))
        if (std::sscanf(v, "%d,%d", &forced_tokens, &forced_splits) != 2 || forced_splits < 1 || forced_splits > steps ||
            (forced_tokens != 256 && forced_tokens != 128 && forced_tokens != 64) || forced_tokens > most)
            forced_tokens = 0;
    double best = 0.0;
    for (int tokens = most; tokens >= 64; tokens /= 2) {
        if (forced_tokens != 0 && tokens != forced_tokens) continue;
        const int64_t m_tiles = (m + tokens - 1) / tokens, tiles = m_tiles * p.n_tiles;
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (forced_tokens != 0) want = forced_splits;
            if (want > 1 && (want > steps / 2 || tiles * want > 1024) && forced_tokens == 0) break;
            const int64_t per = (steps + want - 1) / want, splits = (steps + per - 1) / per, groups = tiles * splits;
            // us of a block, of a round's start and end
            struct Time {
                double block, ends;
            };
            const Time of256 = backward ? Time{2.94, 7.3} : Time{2.74, 4.6}, of128 = backward ? Time{1.88, 4.1} : Time{1.53, 3.5};
            const Time of64 = backward ? Time{2.40, 4.1} : Time{1.85, 2.1}, alone64 = backward ? Time{1.40, 4.1} : Time{1.10, 2.1};
            const auto round = [&](Time t) { return t.block * (double)per + t.ends; };
            double cost = splits > 1 ? 3.8 + (double)(splits * m * cols) * 8 / (backward ? 8.4e6 : 6.1e6) : 0.0;
            if (tokens > 64) {
                cost += (double)((groups + 255) / 256) * round(tokens == 256 ? of256 : of128);
            } else {
                const int64_t rest = groups % 512;
                cost += (double)(groups / 512) * round(of64) + (rest == 0 ? 0.0 : round(rest <= 256 ? alone64 : of64));
            }
            if (best == 0.0 || cost < best) {
                best = cost;
                p.tokens = tokens;
                p.m_tiles = (int)m_tiles;
                p.splits = (int)splits;
                p.steps_per_split = (int)per;
            }
            if (forced_tokens != 0) break;
        }
    }
    p.partial_bytes = p.splits > 1 ? (int64_t)p.splits * m * cols * 4 : 0;
    return p;
}

template <int DT, int GJ, int NW, int P>
static hipError_t launch_ahead(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    const int tiles = NW / p.shares;
    const size_t sums = NW * 4 * 64 * sizeof(float), x = few_x_bytes(a.m < 16 ? a.m : 16, p.steps_per_split), lds = sums > x ? sums : x;
    if (lds > 65536)
        if (hipError_t e = allow_dynamic_lds((const void*)int4_few_kernel<DT, GJ, NW, P>, kInt4FewLds)) return e;
    hipLaunchKernelGGL((int4_few_kernel<DT, GJ, NW, P>), dim3((a.n_tiles + tiles - 1) / tiles, a.splits, p.m_tiles), dim3(64 * NW), lds, s, a);
    return hipGetLastError();
}

template <int DT, int GJ, int NW>
static hipError_t launch_few(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    // (groups of 32 columns: eight blocks ahead would not fit the registers of 16 waves)
    if (GJ > 1 && p.steps_per_split > 4 * p.shares) return launch_ahead<DT, GJ, NW, GJ == 1 ? 4 : 8>(a, p, s);
    return launch_ahead<DT, GJ, NW, 4>(a, p, s);
}

template <int DT, bool WIDE, int C, int GJ>
static hipError_t launch_tile(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    constexpr size_t lds = int4_tile_lds<C, GJ>();
    if (hipError_t e = allow_dynamic_lds((const void*)int4_tile_kernel<DT, WIDE, C, GJ>, lds)) return e;
    hipLaunchKernelGGL((int4_tile_kernel<DT, WIDE, C, GJ>), dim3(p.m_tiles * p.n_tiles * p.splits), dim3(64 * kI4Waves), lds, s, a);
    return hipGetLastError();
}

template <int DT, bool WIDE, int GJ>
static hipError_t launch_forward(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    if (p.few) {
        if (p.waves == 16) return launch_few<DT, GJ, 16>(a, p, s);
        if (p.waves == 8) return launch_few<DT, GJ, 8>(a, p, s);
        return launch_few<DT, GJ, 4>(a, p, s);
    }
    if (p.tokens == 256) return launch_tile<DT, WIDE, 8, GJ>(a, p, s);
    if (p.tokens == 128) return launch_tile<DT, WIDE, 4, GJ>(a, p, s);
    return launch_tile<DT, WIDE, 2, GJ>(a, p, s);
}

template <int DT, bool WIDE, int C>
static hipError_t launch_back(const Int4Args& a, const Int4Plan& p, hipStream_t s) {
    constexpr size_t lds = kI4Ring * int4_back_stage<DT, WIDE, C>() + 4 * kI4Entries * sizeof(uint32_t);
    if (hipError_t e = allow_dynamic_lds((const void*)int4_back_kernel<DT, WIDE, C>, lds)) return e;
    hipLaunchKernelGGL((int4_back_kernel<DT, WIDE, C>), dim3(p.m_tiles * p.n_tiles * p.splits), dim3(64 * kI4Waves), lds, s, a);
    return hipGetLastError();
}

template <int DT, bool WIDE>
static hipError_t launch_typed(const Int4Args& a, const Int4Plan& p, bool backward, hipStream_t s) {
    if (backward) {
        if (p.tokens == 64) return launch_back<DT, WIDE, 2>(a, p, s);
        if (p.tokens == 128) return launch_back<DT, WIDE, 4>(a, p, s);
        return launch_back<DT, WIDE, 8>(a, p, s);
    }
    if (a.group_units % 4 == 0) return launch_forward<DT, WIDE, 4>(a, p, s);
    if (a.group_units % 2 == 0) return launch_forward<DT, WIDE, 2>(a, p, s);
    return launch_forward<DT, WIDE, 1>(a, p, s);
}

hipError_t launch_int4(Int4Args a, const Int4Plan& p, int dtype, bool backward, hipStream_t s) {
    const int cols = backward ? a.k : a.n, sum = backward ? a.n : a.k;
    a.group_mul = (uint32_t)((0x100000000ull + a.group_units - 1) / (uint64_t)a.group_units);
    a.kblocks = (a.k + kI4Block - 1) / kI4Block;
    a.blocks = (sum + 127) / 128;
    a.x_cols = (sum + 7) / 8 * 8;
    a.blocks_per_split = p.steps_per_split;
    a.splits = p.splits;
    a.m_tiles = p.m_tiles;
    a.n_tiles = p.n_tiles;
    a.shares = p.shares;
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
    hipError_t e = dtype == DK_BF16            ? launch_typed<DK_BF16, true>(a, p, backward, s)
                   : a.scale_dtype == DK_FP16 ? launch_typed<DK_FP16, false>(a, p, backward, s)
                                              : launch_typed<DK_FP16, true>(a, p, backward, s);
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL(int4_join_kernel, dim3((cols + 1023) / 1024, a.m < 4096 ? a.m : 4096), dim3(256), 0, s, a, cols);
    return hipGetLastError();
}

}  // namespace dk
