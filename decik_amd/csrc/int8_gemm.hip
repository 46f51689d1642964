// Product of 8-bit integer matrices with a scale per token and per channel, on 32x32x32 integer MFMAs:
//   forward:   y[m, n]  = (sum_k xq[m, k] wq[n, k]) xs[m] ws[n] + bias[n]
//   TR:        y[m, n]  = (sum_k xq[m, k] wq[k, n]) xs[m]         (the input gradient: xq holds the
//              gradient times the channel scales, quantized per token; wq as it is stored)
// Sums are exact in 32-bit integers (k <= 131071), so neither the order nor the split of k changes a
// result; the scales are applied in fp32 and rounded once.
//
// Work-group: tiles of 256, 128 or 64 tokens by 256 channels (eight waves) or 64 by 64 (four), steps of 128
// along k. Both operands go straight to LDS (16 bytes a lane) through a ring of stages; one wait and one
// barrier a step, before its last part, so that the next step's first operands are read behind MFMAs too.
// Rows of a stage are 128 bytes, their 16-byte chunks permuted by row so that the operand reads (32 rows at
// one chunk) spread over the banks. TR stages wq as it lies (rows along k, a row of the tile's channels each)
// and turns it through the transposed LDS read of 8-bit elements: in each 16 lanes, lanes 2 r and 2 r + 1
// read the 16 bytes of row r, lane i receives byte i of the 8 rows.
//
// Bound: at [8192, 18944] x 3584 the forward takes 504 to 541 us from GPU to GPU (2.06 to 2.21 POP/s), the input
// gradient 474 to 512 (2.17 to 2.35); torch's library product of the same sizes, without scales, 514 to 616 and
// 569 to 571. Matrix cores are busy 59 and 62% of the cycles, at 1.7 GHz under this load. On the GPU of 541 and
// 512 us, timing copies without the loads of the loop took 480 and 430, without the operand reads 550 and 550,
// without either 440 and 380: the loads cost most, through their issue and the L2's bandwidth (64 KB a step and
// CU), not through latency (lines touched a step or more ahead in the L2 made it 3 to 8% slower).
// The last round of tiles is 7 to 12% idle. Also measured, not kept: tiles of 128 by 128 on four waves, two
// work-groups a CU (equal or slower everywhere), operand reads pinned before the MFMAs (+0 to 5%), bands of
// four token tiles (equal).
#include "elem.h"
#include "gemm_common.h"

namespace dk {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int int2v_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const uint8_t* lds_t;
typedef int int16v_t __attribute__((ext_vector_type(16)));

constexpr int kI8BK = 128;

// tiles of TM = 256, 128 or 64 tokens by BN = 256 channels (eight waves), or 64 by 64 (four)
__host__ __device__ constexpr int i8_waves(int bn) { return bn == 256 ? 8 : 4; }
__host__ __device__ constexpr int i8_stage_bytes(int tm, int bn) { return (bn + tm) * kI8BK; }
__host__ __device__ constexpr int i8_stages(int tm, int bn) {
    return bn == 64 ? 4 : tm == 256 ? 2 : 3;
}
__host__ __device__ constexpr size_t i8_lds(int tm, int bn) {  // with the channels' scales and biases
    return (size_t)i8_stages(tm, bn) * i8_stage_bytes(tm, bn) + 8 * bn;
}

// chunk permutation of a row: tokens are read 32 consecutive rows at a time
__device__ __forceinline__ int row_key(int r) { return (r >> 1) & 7; }

__device__ __forceinline__ int4_t bload128i(rsrc_t r, uint32_t off) {
    const u32x4_t v = bload128(r, off);
    return __builtin_bit_cast(int4_t, v);
}

__device__ __forceinline__ int4_t lds128(const uint8_t* p) { return *(const int4_t*)p; }

// Operands from a TR stage: 16 rows of a lane's byte column, two transposed reads of 8 rows each. One asm
// block with its own wait: the builtin counts as aliasing every load to LDS in flight and would drain the
// ring at every read. R8: bytes of 8 rows; the next slice is 4 R8 on.
template <int R8>
__device__ __forceinline__ void lds_tr8(const uint8_t* st, const uint32_t (&at)[2], int4_t (&o)[1][2]) {
    int2v_t a, b, c, d;
    asm volatile(
        "ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %4 offset:%6\n\t"
        "ds_read_b64_tr_b8 %2, %5\n\tds_read_b64_tr_b8 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
        : "v"((lds_t)(st + at[0])), "v"((lds_t)(st + at[1])), "n"(R8)
        : "memory");
    o[0][0] = int4_t{a.x, a.y, b.x, b.y};
    o[0][1] = int4_t{c.x, c.y, d.x, d.y};
}
template <int R8>
__device__ __forceinline__ void lds_tr8(const uint8_t* st, const uint32_t (&at)[2], int4_t (&o)[2][2]) {
    int2v_t a, b, c, d, e, f, g, h;
    asm volatile(
        "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %8 offset:%10\n\t"
        "ds_read_b64_tr_b8 %2, %9\n\tds_read_b64_tr_b8 %3, %9 offset:%10\n\t"
        "ds_read_b64_tr_b8 %4, %8 offset:%11\n\tds_read_b64_tr_b8 %5, %8 offset:%12\n\t"
        "ds_read_b64_tr_b8 %6, %9 offset:%11\n\tds_read_b64_tr_b8 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(e), "=&v"(f), "=&v"(g), "=&v"(h)
        : "v"((lds_t)(st + at[0])), "v"((lds_t)(st + at[1])), "n"(R8), "n"(4 * R8), "n"(5 * R8)
        : "memory");
    o[0][0] = int4_t{a.x, a.y, b.x, b.y};
    o[0][1] = int4_t{c.x, c.y, d.x, d.y};
    o[1][0] = int4_t{e.x, e.y, f.x, f.y};
    o[1][1] = int4_t{g.x, g.y, h.x, h.y};
}
template <int R8>
__device__ __forceinline__ void lds_tr8(const uint8_t* st, const uint32_t (&at)[1], int4_t (&o)[4][1]) {
    int2v_t a, b, c, d, e, f, g, h;
    asm volatile(
        "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %8 offset:%9\n\t"
        "ds_read_b64_tr_b8 %2, %8 offset:%10\n\tds_read_b64_tr_b8 %3, %8 offset:%11\n\t"
        "ds_read_b64_tr_b8 %4, %8 offset:%12\n\tds_read_b64_tr_b8 %5, %8 offset:%13\n\t"
        "ds_read_b64_tr_b8 %6, %8 offset:%14\n\tds_read_b64_tr_b8 %7, %8 offset:%15\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(e), "=&v"(f), "=&v"(g), "=&v"(h)
        : "v"((lds_t)(st + at[0])), "n"(R8), "n"(4 * R8), "n"(5 * R8), "n"(8 * R8), "n"(9 * R8), "n"(12 * R8),
          "n"(13 * R8)
        : "memory");
    o[0][0] = int4_t{a.x, a.y, b.x, b.y};
    o[1][0] = int4_t{c.x, c.y, d.x, d.y};
    o[2][0] = int4_t{e.x, e.y, f.x, f.y};
    o[3][0] = int4_t{g.x, g.y, h.x, h.y};
}

template <int V>
struct Int {
    static constexpr int value = V;
};

// chunk permutation of a TR stage's row r (along k): the eight rows of a transposed read, at one chunk or at
// two neighbouring ones, spread over the banks
template <int BN>
__device__ __forceinline__ int tr_key(int r) {
    return ((r & 7) / (256 / BN)) << 1;
}

template <int TM, int BN, bool TR>
struct I8Tile {
    static constexpr int NW = i8_waves(BN);
    // waves along channels and tokens
    static constexpr int WN = BN == 256 ? (TM == 256 ? (TR ? 4 : 2) : TM == 128 ? 4 : 8) : 2;
    static constexpr int WM = NW / WN;
    static constexpr int TN = BN / WN / 32, TT = TM / WM / 32;  // 32x32 blocks a wave
    static constexpr int WLOADS = BN * kI8BK / 1024 / NW, XLOADS = TM * kI8BK / 1024 / NW;  // a wave and step
    static constexpr int LOADS = WLOADS + XLOADS;
    // slices whose operands are read at once, ahead of the MFMAs: small tiles have few MFMAs a slice to hide
    // the reads behind
    static constexpr int U = TM == 256 ? 1 : TM == 128 ? 2 : 4;
};

template <int OUT>
__device__ __forceinline__ void store4(typename Elem<OUT>::type* p, float4_t v, int left) {
    typedef typename Elem<OUT>::type E;
    typedef E vec4 __attribute__((ext_vector_type(4)));
    typedef vec4 loose4 __attribute__((aligned(sizeof(E))));
    if (left >= 4) {
        *(loose4*)p = __builtin_convertvector(v, vec4);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) p[e] = (E)v[e];
    }
}

__device__ __forceinline__ int4_t quad(const int16v_t& v, int q) {
    return int4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
}

// four sums times the token's scale and (not TR) the channels' scales, plus their biases (BN on)
template <bool TR, int BN>
__device__ __forceinline__ float4_t scaled(int4_t v, float xs, const float* chan) {
    float4_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)v[e] * xs;
    if constexpr (!TR) f = f * *(const float4_t*)chan + *(const float4_t*)(chan + BN);
    asm("" : "+v"(f));  // keeps the products out of mixed-precision multiply-adds
    return f;
}

// OUT: an element type, or -1 for the int32 partial sums of a split
template <int TM, int BN, bool TR, int OUT>
__global__ __launch_bounds__(64 * i8_waves(BN), 2) void int8_gemm_kernel(const Int8GemmArgs a) {
    typedef I8Tile<TM, BN, TR> T;
    constexpr int S = i8_stages(TM, BN), STAGE = i8_stage_bytes(TM, BN);
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, g = lane >> 5;

    // consecutive tiles on one XCD (work-groups are dealt to the eight in turn), token tiles fastest
    // within groups of eight, so that the tiles of an XCD at one time share rows of both operands
    const int per = a.m_tiles * a.n_tiles, nwg = per * a.splits;
    const int xcd = blockIdx.x & 7, r8 = nwg & 7;
    const int L = xcd * (nwg >> 3) + min(xcd, r8) + (blockIdx.x >> 3);
    const int split = L / per, tile = L - split * per;
    const int band = tile / (8 * a.n_tiles), in = tile - band * 8 * a.n_tiles;
    const int rows = min(8, a.m_tiles - 8 * band);
    const int m0 = (8 * band + in % rows) * TM, n0 = (in / rows) * BN;
    const int k_begin = split * a.steps_per_split * kI8BK;
    const int steps = min(a.steps_per_split, (a.k + kI8BK - 1) / kI8BK - split * a.steps_per_split);
    const int kpad = (a.k + 15) & ~15, npad = (a.n + 15) & ~15;

    const int8_t* const xb = a.x + (int64_t)m0 * a.ldx;
    const uint32_t x_bytes = (uint32_t)((min(TM, a.m - m0) - 1) * a.ldx + kpad);
    const int8_t* const wb = TR ? a.w + n0 : a.w + (int64_t)n0 * a.ldw;
    const uint32_t w_bytes = TR ? (uint32_t)min(BN, npad - n0)
                                : (uint32_t)((min(BN, a.n - n0) - 1) * a.ldw + kpad);

    // this lane's source offsets, and its column along k, of every load of a step
    uint32_t woff[T::WLOADS], xoff[T::XLOADS];
    int wcol[T::WLOADS], xcol[T::XLOADS];
#pragma unroll
    for (int i = 0; i < T::WLOADS; ++i) {
        const int q = wave * T::WLOADS + i;
        if constexpr (TR) {
            constexpr int CHUNKS = BN / 16;
            const int r = 64 / CHUNKS * q + lane / CHUNKS;
            wcol[i] = 0;
            woff[i] = r * (uint32_t)a.ldw + 16 * ((lane % CHUNKS) ^ tr_key<BN>(r));
        } else {
            const int r = 8 * q + (lane >> 3);
            wcol[i] = 16 * ((lane & 7) ^ row_key(r));
            woff[i] = r * (uint32_t)a.ldw + wcol[i];
        }
    }
#pragma unroll
    for (int i = 0; i < T::XLOADS; ++i) {
        const int r = 8 * (wave * T::XLOADS + i) + (lane >> 3);
        xcol[i] = 16 * ((lane & 7) ^ row_key(r));
        xoff[i] = r * (uint32_t)a.ldx + xcol[i];
    }

    // where the loads of step t come from and go to; past the last step they read nothing (and write zeros
    // nobody reads), which keeps the number of loads in flight the same for every wait
    struct Source {
        rsrc_t w, x;
        uint8_t* stage;
        int left;
    };
    const auto source = [&](int t) {
        const int k0 = k_begin + t * kI8BK;
        const bool live = t < steps;
        Source f;
        f.stage = smem + (t % S) * STAGE;
        f.left = live ? a.k - k0 : 0;
        f.x = make_rsrc(xb + k0, live ? x_bytes - (uint32_t)k0 : 0u);
        if constexpr (TR)
            f.w = make_rsrc(wb + (int64_t)k0 * a.ldw,
                            live ? (uint32_t)(min(kI8BK, f.left) - 1) * (uint32_t)a.ldw + w_bytes : 0u);
        else
            f.w = make_rsrc(wb + k0, live ? w_bytes - (uint32_t)k0 : 0u);
        return f;
    };
    const auto fetch = [&](const Source& f, int i) {
        if (i < T::WLOADS) {
            bload128_lds(f.w, f.stage + 1024 * (wave * T::WLOADS + i), TR ? woff[i] : off_if(wcol[i] < f.left, woff[i]));
        } else {
            const int x = i - T::WLOADS;
            bload128_lds(f.x, f.stage + BN * kI8BK + 1024 * (wave * T::XLOADS + x),
                         off_if(xcol[x] < f.left, xoff[x]));
        }
    };

    int16v_t acc[T::TN][T::TT];
#pragma unroll
    for (int i = 0; i < T::TN; ++i)
#pragma unroll
        for (int j = 0; j < T::TT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    const int wn = (wave / T::WM) * 32 * T::TN, wm = (wave % T::WM) * 32 * T::TT;
    // this lane's operand addresses in a stage, for chunk pair 0 (slice s flips bits of the chunk)
    uint32_t wat[T::TN], xat[T::TT];
#pragma unroll
    for (int i = 0; i < T::TN; ++i) {
        if constexpr (TR) {
            const int r = (lane & 15) >> 1, c = (wn + 32 * i) / 16 + ((lane >> 4) & 1);
            wat[i] = (16 * g + r) * BN + 16 * (c ^ tr_key<BN>(r)) + 8 * (lane & 1);
        } else {
            const int r = wn + 32 * i + l32;
            wat[i] = r * 128 + 16 * (g ^ row_key(r));
        }
    }
#pragma unroll
    for (int j = 0; j < T::TT; ++j) {
        const int r = wm + 32 * j + l32;
        xat[j] = BN * kI8BK + r * 128 + 16 * (g ^ row_key(r));
    }

    // operands of U slices (32 of k each) of a stage: parts 0 .. 4 / U - 1 of step t
    constexpr int U = T::U;
    struct Part {
        int4_t w[U][T::TN], x[U][T::TT];
    };
    const auto read = [&](Part& f, int t, int part) {
        const uint8_t* const st = smem + (t % S) * STAGE;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = part * U + u;
#pragma unroll
            for (int j = 0; j < T::TT; ++j) f.x[u][j] = lds128(st + (xat[j] ^ (32 * s)));
            if constexpr (!TR) {
#pragma unroll
                for (int i = 0; i < T::TN; ++i) f.w[u][i] = lds128(st + (wat[i] ^ (32 * s)));
            }
        }
        if constexpr (TR) lds_tr8<8 * BN>(st + part * U * 32 * BN, wat, f.w);
    };
    // The MFMAs of a part, and between them loads `from` .. `to` - 1 of a coming step: issued at once, the loads
    // of eight waves fill the address queue and hold up the MFMAs behind them ([830, 8960] x 1536 19.3 against
    // 17.3 us; the 64-token tiles, whose part is a whole step, take them at once: 26.5 against 27.0 at
    // [830, 1536] x 8960). On the largest tiles the wave that multiplies goes first (8192 tokens 562 -> 548 us;
    // 128-token tiles are slower with it).
    const auto multiply = [&](const Part& f, const Source& next, int from, int to) {
        if constexpr (TM == 256) __builtin_amdgcn_s_setprio(1);
        if constexpr (U == 4) {
#pragma unroll
            for (int i = from; i < to; ++i) fetch(next, i);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < T::TN; ++i)
#pragma unroll
                for (int j = 0; j < T::TT; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[u][i], f.x[u][j], acc[i][j], 0, 0, 0);
                    const int n = (u * T::TN + i) * T::TT + j;  // of eight
                    if (U != 4 && n % 2 == 0 && from + n / 2 < to) {
                        fetch(next, from + n / 2);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
        if constexpr (TM == 256) __builtin_amdgcn_s_setprio(0);
    };

    // the tile's channel scales and biases
    float* const chan = (float*)(smem + S * STAGE);
    if constexpr (!TR && OUT >= 0) {
        const int c = threadIdx.x % BN, n = n0 + c;
        if (threadIdx.x < 2 * BN) {
            float v = 0.0f;
            if (n < a.n) {
                if (threadIdx.x < BN) v = a.ws[n];
                else if (a.bias != nullptr) v = load_any(a.bias, a.bias_dtype, n);
            }
            chan[threadIdx.x] = v;
        }
    }

    // loads of step t + S issued in part p of steps t (after its barrier: the last part) and t + 1
    constexpr int PARTS = 4 / U;
    constexpr int FIRST = PARTS == 1 ? T::LOADS : PARTS == 2 ? (T::LOADS + 1) / 2 : 4;
    static_assert(T::LOADS <= FIRST * PARTS && (PARTS == 1 || FIRST <= 4), "loads of a step");
    Part f[2];
#pragma unroll
    for (int t = 0; t < S - 1; ++t) {
        const Source next = source(t);
#pragma unroll
        for (int i = 0; i < T::LOADS; ++i) fetch(next, i);
    }
    Source next = source(S - 1);
#pragma unroll
    for (int i = 0; i < FIRST; ++i) fetch(next, i);
    wait_vmcnt<T::LOADS * (S - 2) + FIRST>();
    lds_barrier();
    read(f[0], 0, 0);
    // a step whose first part is in f[P]
    const auto step = [&](int t, auto parity) {
        constexpr int P = decltype(parity)::value;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const int now = (P + part) & 1;
            if (part + 1 < PARTS) {
                read(f[now ^ 1], t, part + 1);
                multiply(f[now], next, min(FIRST * (part + 1), T::LOADS), min(FIRST * (part + 2), T::LOADS));
            } else {
                // every wave has read the last of this stage: it is free, and the next one is whole
                wait_vmcnt<T::LOADS * (S - 2)>();
                lds_barrier();
                next = source(t + S);
                read(f[now ^ 1], t + 1, 0);
                multiply(f[now], next, 0, FIRST);
            }
        }
    };
    if constexpr (U == 4) {
        int t = 0;
        for (; t + 1 < steps; t += 2) {
            step(t, Int<0>());
            step(t + 1, Int<1>());
        }
        if (t < steps) step(t, Int<0>());
    } else {
        for (int t = 0; t < steps; ++t) step(t, Int<0>());
    }
    wait_vmcnt<0>();
    lds_barrier();

    // lane: token wm + 32 j + l32, channels wn + 32 i + 8 q + 4 g + 0..3
    if constexpr (OUT < 0 || OUT == DK_FP32) {
#pragma unroll
        for (int j = 0; j < T::TT; ++j) {
            const int m = m0 + wm + 32 * j + l32;
            if (m >= a.m) continue;
            const float xs = OUT < 0 ? 0.0f : a.xs[m];
#pragma unroll
            for (int i = 0; i < T::TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = wn + 32 * i + 8 * q + 4 * g, n = n0 + c;
                    if (n >= a.n) continue;
                    const int4_t v = quad(acc[i][j], q);
                    if constexpr (OUT < 0)  // slab rows are padded to four channels
                        *(int4_t*)(a.partials + (int64_t)split * a.slab + (int64_t)m * a.ldp + n) = v;
                    else
                        store4<DK_FP32>((float*)a.y + (int64_t)m * a.ldy + n, scaled<TR, BN>(v, xs, chan + c), a.n - n);
                }
        }
    } else {
        // 16-bit outputs leave as whole rows: 32 tokens of the wave's channels at a time through LDS
        typedef typename Elem<OUT>::type E;
        constexpr int ROW = 64 * T::TN + 16;  // bytes
        constexpr int LANES = 4 * T::TN;      // lanes a row of 16-byte pieces
        uint8_t* const stage = smem + wave * 32 * ROW;
#pragma unroll
        for (int j = 0; j < T::TT; ++j) {
            const int mrow = m0 + wm + 32 * j;
            const float xs = mrow + l32 < a.m ? a.xs[mrow + l32] : 0.0f;
#pragma unroll
            for (int i = 0; i < T::TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = 32 * i + 8 * q + 4 * g;
                    const float4_t v = scaled<TR, BN>(quad(acc[i][j], q), xs, chan + wn + c);
                    store4<OUT>((E*)(stage + l32 * ROW) + c, v, 4);
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = 0; r < 32; r += 64 / LANES) {
                const int row = r + lane / LANES, c = 8 * (lane % LANES), n = n0 + wn + c, m = mrow + row;
                const typename Elem<OUT>::vec v = *(const typename Elem<OUT>::vec*)(stage + row * ROW + 2 * c);
                if (m >= a.m || n >= a.n) continue;
                E* const y = (E*)a.y + (int64_t)m * a.ldy + n;
                if (n + 8 <= a.n && a.past_caches) {
                    __builtin_nontemporal_store(v, (typename Elem<OUT>::loose*)y);
                } else if (n + 8 <= a.n) {
                    *(typename Elem<OUT>::loose*)y = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n + e < a.n) y[e] = v[e];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Split sums added, scaled, rounded: four channels a thread.
template <int OUT>
__global__ __launch_bounds__(256) void int8_reduce_kernel(const Int8GemmArgs a) {
    const int quads = a.ldp / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.m * quads) return;
    const int m = (int)(i / quads), n = 4 * (int)(i - (int64_t)m * quads);
    int4_t v = {0, 0, 0, 0};
    for (int s = 0; s < a.splits; ++s) v += *(const int4_t*)(a.partials + s * a.slab + (int64_t)m * a.ldp + n);
    const float xs = a.xs[m];
    const int left = a.n - n;
    float4_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[e] = (float)v[e] * xs;
        if (a.ws != nullptr && e < left) f[e] *= a.ws[n + e];
        if (a.bias != nullptr && e < left) f[e] += load_any(a.bias, a.bias_dtype, n + e);
    }
    store4<OUT>((typename Elem<OUT>::type*)a.y + (int64_t)m * a.ldy + n, f, left);
}

// ---- quantization of rows ------------------------------------------------------------------------
// scale = absmax / 127, q = rint(x * (127 / absmax)) in fp32 (COL: of x times a scale per column). Rows
// whose largest magnitude is below 2^-120 count as zeros; a row that holds an infinity or NaN gets the
// scale NaN and zeros, so that its products are NaN. THREADS threads a row, which stays in their registers
// between its maximum and its rounding (R groups of eight a thread), or is read again (R = 0).
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// eight columns of a row, zeros past the last
template <int DT>
__device__ __forceinline__ typename Elem<DT>::vec quant_load(const Int8QuantArgs& a, int64_t row, int col) {
    const typename Elem<DT>::type* p = (const typename Elem<DT>::type*)a.x + row * a.ldx + col;
    if (col + 8 <= a.k) return load8_raw<DT>(p);
    typename Elem<DT>::vec v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < a.k) v[e] = p[e];
    return v;
}

__device__ __forceinline__ float8_t scale_load(const float* s, int col, int k) {
    if (col + 8 <= k) return load8<DK_FP32>(s + col);
    float8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < k) v[e] = s[col + e];
    return v;
}

__device__ __forceinline__ uint32_t top8(float8_t v, uint32_t top) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[e]));
    return top;
}

// Eight values rounded to integers (to nearest even, |v inv| <= 127): in the sum with 1.5 * 2^23 the fp32 unit
// is 1, so the addition rounds and the low byte holds the integer in two's complement.
__device__ __forceinline__ u32x2_t quant8(float8_t v, float inv) {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(v[e] * inv + 12582912.0f);
    u32x2_t o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000c0cu);
        o[h] = lo | hi;
    }
    return o;
}

// scale of a row with the largest magnitude `top` (its bits), and what its values are multiplied by (0: zeros)
__device__ __forceinline__ void quant_scale(uint32_t top, float& inv, float& scale) {
    const float most = __uint_as_float(top);
    const bool bad = top >= 0x7F800000u, none = most < 7.523163845262640e-37f;  // 2^-120
    inv = bad || none ? 0.0f : 127.0f / most;
    scale = bad ? __builtin_nanf("") : none ? 0.0f : most / 127.0f;
}

// The row stays in registers between its maximum and its rounding (R groups of eight a thread), or is read
// again (R = 0). THREADS threads a row. Bound: HBM, at [8192, 18944] fp16 with column scales 97 to 107 us (4.8 to
// 4.35 TB/s; a large copy reaches 5.2), [8192, 3584] 18.1. Several rows a work-group, the column scales read once
// for them, were slower (175 and 25.7 us beside 107 and 18.3: fewer waves).
template <int DT, bool COL, int THREADS, int R>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void int8_quantize_kernel(const Int8QuantArgs a) {
    constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, ROWS = BLOCK / THREADS, NW = THREADS / 64;
    __shared__ uint32_t tops[NW];
    const int tid = threadIdx.x % THREADS;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
    if (THREADS == 64 && row >= a.rows) return;  // whole waves; larger groups have one row a work-group
    const int groups = (a.k + 7) / 8, padded = (a.k + 15) / 16 * 2;
    const auto load = [&](int q) {
        const float8_t v = widen8<DT>(quant_load<DT>(a, row, 8 * q));
        return COL ? v * scale_load(a.col_scale, 8 * q, a.k) : v;
    };
    float8_t v[R > 0 ? R : 1];
    uint32_t top = 0;
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int q = tid + i * THREADS;
            if (q < groups) v[i] = load(q);
            else v[i] = float8_t{0, 0, 0, 0, 0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < R; ++i) top = top8(v[i], top);
    } else {
        for (int q = tid; q < groups; q += THREADS) top = top8(load(q), top);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) top = max(top, tops[i]);
    }
    float inv, scale;
    quant_scale(top, inv, scale);
    if (tid == 0) a.scale[row] = scale;
    int8_t* const out = a.q + row * a.ldq;
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int q = tid + i * THREADS;
            if (q < padded) *(u32x2_t*)(out + 8 * q) = inv == 0.0f ? u32x2_t{0, 0} : quant8(v[i], inv);
        }
    } else {
        for (int q = tid; q < padded; q += THREADS) {
            const float8_t x = q < groups ? load(q) : float8_t{0, 0, 0, 0, 0, 0, 0, 0};
            *(u32x2_t*)(out + 8 * q) = inv == 0.0f ? u32x2_t{0, 0} : quant8(x, inv);
        }
    }
}

template <int DT, bool COL>
static void launch_quantize_typed(const Int8QuantArgs& a, hipStream_t s) {
    const int groups = (a.k + 15) / 16 * 2;
    const unsigned rows = (unsigned)a.rows;
    if (groups <= 64 * 4)
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 64, 4>), dim3((rows + 3) / 4), dim3(256), 0, s, a);
    else if (groups <= 256 * 2)
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 256, 2>), dim3(rows), dim3(256), 0, s, a);
    else if (groups <= 256 * 4)
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 256, 4>), dim3(rows), dim3(256), 0, s, a);
    else if (groups <= 512 * 3)
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 512, 3>), dim3(rows), dim3(512), 0, s, a);
    else if (groups <= 512 * 5)
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 512, 5>), dim3(rows), dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((int8_quantize_kernel<DT, COL, 512, 0>), dim3(rows), dim3(512), 0, s, a);
}

hipError_t launch_int8_quantize(const Int8QuantArgs& a, int dtype, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    const bool col = a.col_scale != nullptr;
    if (dtype == DK_FP16)
        col ? launch_quantize_typed<DK_FP16, true>(a, s) : launch_quantize_typed<DK_FP16, false>(a, s);
    else if (dtype == DK_BF16)
        col ? launch_quantize_typed<DK_BF16, true>(a, s) : launch_quantize_typed<DK_BF16, false>(a, s);
    else
        col ? launch_quantize_typed<DK_FP32, true>(a, s) : launch_quantize_typed<DK_FP32, false>(a, s);
    return hipGetLastError();
}

// Few tokens: the weight streams from memory once, straight to registers. A work-group of WAVES waves
// owns 16 channels, the waves take slices of k; 16x16x64 integer MFMAs with MT blocks of 16 tokens (rows
// past m repeat the last one and are dropped), U 64-byte columns of the weight in flight a wave. The exact
// integer sums of the waves meet in LDS. Bound by the weight's stream from memory and, as the tokens grow,
// by the reads of x, which every work-group makes: [18944, 3584] with the weight from memory 18.3 us at one
// token, 22.2 at 8, 35 at 32 with the quantizer's launch (its 68 MB alone take 13 us). Measured and not
// kept: 32 and 64 channels a work-group (21 - 25 us at one token; 32 at 32 tokens), columns loaded one by one
// as they are used up (+1 us), non-temporal loads (+0 to 2 us).
template <int MT, int WAVES, int OUT>
__global__ __launch_bounds__(64 * WAVES) void int8_few_kernel(const Int8GemmArgs a) {
    constexpr int U = 8;
    __shared__ int red[WAVES][MT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = 16 * blockIdx.x, l16 = lane & 15, c = 16 * (lane >> 4);
    const int cols = (a.k + 63) / 64, share = (cols + WAVES - 1) / WAVES;
    const int begin = wave * share, end = min(cols, begin + share);
    // buffers of this work-group's channels and of x: offsets past a row's k read zeros
    const int kpad = (a.k + 15) & ~15;
    const rsrc_t wr = make_rsrc(a.w + (int64_t)n0 * a.ldw, (uint32_t)((min(16, a.n - n0) - 1) * a.ldw + kpad));
    const rsrc_t xr = make_rsrc(a.x, (uint32_t)((a.m - 1) * a.ldx + kpad));
    const uint32_t woff = l16 * (uint32_t)a.ldw + c;
    uint32_t xoff[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xoff[t] = min(16 * t + l16, a.m - 1) * (uint32_t)a.ldx + c;
    int4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = int4_t{0, 0, 0, 0};
    const int last = min(64 * end, a.k) - c;
    for (int b = begin; b < end; b += U) {
        int4_t wf[U], xf[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = off_if(64 * (b + u) < last, 64u * (b + u));
            wf[u] = bload128i(wr, woff + at);
#pragma unroll
            for (int t = 0; t < MT; ++t) xf[u][t] = bload128i(xr, xoff[t] + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][t], acc[t], 0, 0, 0);
    }
    // lane: channels 4 (lane / 16) + 0..3 of token l16
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][t][l16 * 16 + 4 * (lane >> 4) + e] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * MT; i += 64 * WAVES) {
        const int m = i >> 4, n = n0 + (i & 15);
        if (m >= a.m || n >= a.n) continue;
        int v = 0;
#pragma unroll
        for (int s = 0; s < WAVES; ++s) v += red[s][m >> 4][i & 255];
        float f = (float)v * a.xs[m] * a.ws[n];
        if (a.bias != nullptr) f += load_any(a.bias, a.bias_dtype, n);
        store1<OUT>((typename Elem<OUT>::type*)a.y + (int64_t)m * a.ldy + n, f);
    }
}

// The same with x as it comes (fp16, bf16 or fp32): every work-group quantizes the few rows for itself
// (they come from the L2) into LDS while its first weights are on their way, which saves the launch of the
// quantizer and its round trip. Weights from memory: [18944, 3584] at one token 16.0 us (4.2 TB/s) against 18.3,
// [3584, 3584] 6.0 against 8.4; at two tokens equal, at four 22.0 against 19.8. A repeated [18944, 3584] (68 MB) is
// read from the last cache: 14.4.
template <int DT, int WAVES, int OUT>
__global__ __launch_bounds__(64 * WAVES) void int8_few_fused_kernel(const Int8GemmArgs a, const Int8QuantArgs q) {
    constexpr int U = 8;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ int red[WAVES][256];
    __shared__ uint32_t tops[WAVES];
    __shared__ float scales[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = 16 * blockIdx.x, l16 = lane & 15, c = 16 * (lane >> 4);
    const int cols = (a.k + 63) / 64, share = (cols + WAVES - 1) / WAVES;
    const int begin = wave * share, end = min(cols, begin + share);
    const int kpad = (a.k + 15) & ~15;
    const rsrc_t wr = make_rsrc(a.w + (int64_t)n0 * a.ldw, (uint32_t)((min(16, a.n - n0) - 1) * a.ldw + kpad));
    const uint32_t woff = l16 * (uint32_t)a.ldw + c;
    const int last = min(64 * end, a.k) - c;
    int4_t wf[U];
    const auto fetch = [&](int b) { return bload128i(wr, woff + off_if(64 * b < last, 64u * b)); };
#pragma unroll
    for (int u = 0; u < U; ++u) wf[u] = fetch(begin + u);
    const int ld = 64 * cols, groups = ld / 8;  // LDS rows, zeros past k
    for (int m = 0; m < a.m; ++m) {
        uint32_t top = 0;
        for (int g = threadIdx.x; 8 * g < a.k; g += 64 * WAVES) top = top8(widen8<DT>(quant_load<DT>(q, m, 8 * g)), top);
#pragma unroll
        for (int o = 1; o < 64; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        if (lane == 0) tops[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = max(top, tops[i]);
        float inv, scale;
        quant_scale(top, inv, scale);
        if (threadIdx.x == 0) scales[m] = scale;
        for (int g = threadIdx.x; g < groups; g += 64 * WAVES) {
            float8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
            if (8 * g < a.k) v = widen8<DT>(quant_load<DT>(q, m, 8 * g));
            *(u32x2_t*)(smem + m * ld + 8 * g) = inv == 0.0f ? u32x2_t{0, 0} : quant8(v, inv);
        }
        __syncthreads();
    }
    const uint8_t* const x = smem + min(l16, a.m - 1) * ld + c;
    int4_t acc = {0, 0, 0, 0};
    for (int b = begin; b < end; b += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b + u >= end) break;
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], lds128(x + 64 * (b + u)), acc, 0, 0, 0);
            wf[u] = fetch(b + u + U);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][l16 * 16 + 4 * (lane >> 4) + r] = acc[r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * a.m; i += 64 * WAVES) {
        const int m = i >> 4, n = n0 + (i & 15);
        if (n >= a.n) continue;
        int v = 0;
#pragma unroll
        for (int s = 0; s < WAVES; ++s) v += red[s][i];
        float f = (float)v * scales[m] * a.ws[n];
        if (a.bias != nullptr) f += load_any(a.bias, a.bias_dtype, n);
        store1<OUT>((typename Elem<OUT>::type*)a.y + (int64_t)m * a.ldy + n, f);
    }
}

// ---- launches ------------------------------------------------------------------------------------

static Int8Plan make_plan(int64_t m, int64_t n, int64_t k, int cus, bool tr) {
    Int8Plan best{};
    const int64_t steps = (k + kI8BK - 1) / kI8BK > 0 ? (k + kI8BK - 1) / kI8BK : 1;
    double best_us = 0;
    // Estimated time of a launch, fitted to 170 timed launches (17 sizes of 64 to 8192 tokens and summed axes of 1121
    // to 18944, both ways, every tile, 1 to 15 splits; root mean square of the deviation 8%; its choice within 3% of
    // the best of each size but one, 6%; on shorter sums it extrapolates: [8192, 8960] x 384 86 us, measured 63,
    // [8192, 3584] x 512 39 and 29): rounds of work-groups of a number of steps each, whose time grows from `light`
    // to `full` with the share of the CUs that work, and a last part; sums of splits written and read back.
    struct Tile {
        int tm, bn;
        double light, full, last;
    };
    const Tile tiles[4] = {{256, 256, 0.99, 1.46, 5.0}, {128, 256, 0.51, 0.91, 2.8}, {64, 256, 0.42, 0.63, 1.8},
                           {64, 64, 0.22, 0.24, 0.2}};
    for (const Tile& v : tiles) {
        const int64_t mt = (m + v.tm - 1) / v.tm, nt = (n + v.bn - 1) / v.bn;
        for (int64_t sp = 1; sp <= steps && sp <= 32; ++sp) {
            const int64_t sps = (steps + sp - 1) / sp;
            if ((steps + sps - 1) / sps != sp) continue;
            const int64_t wgs = mt * nt * sp, rounds = (wgs + cus - 1) / cus, sums = sp * m * ((n + 3) / 4 * 4);
            if (sp > 1 && sums > (int64_t(1) << 28)) continue;
            const double load = wgs < cus ? (double)wgs / cus : 1.0;
            double us = 2.5 + rounds * (sps * (v.light + (v.full - v.light) * load) + v.last) + m * n * 0.5e-6;
            if (sp > 1) us += 3.9 + sums * 1.5e-6;
            if (best_us == 0 || us < best_us) {
                best_us = us;
                best.tm = v.tm;
                best.bn = v.bn;
                best.m_tiles = (int)mt;
                best.n_tiles = (int)nt;
                best.splits = (int)sp;
                best.steps_per_split = (int)sps;
                best.partial_bytes = sp > 1 ? sums * 4 : 0;
            }
        }
    }
    // Few tokens: the streaming kernel where its estimate is the smaller one, weights from memory on both sides
    // (the tiles' estimate knows them in the caches). Measured, streaming / tiles, us: [3584, 3584] 9.1 / 12.0
    // at 8 tokens, 11.1 / 12.2 at 32; [8960, 1536] 9.4 / 9.6 and 13.5 / 10.2; [18944, 3584] 22.3 / 21.4 and 35.1
    // / 23.2; [3584] x 18944 27.0 / 23.3 at 8; [512] x 3584 7.9 / 10.0 and 10.3 / 10.6.
    const double few_us = 6.5 + n * k / 5.5e6 + m * n * k * 7.9e-9 + k * 3e-4;
    if (!tr && m <= kInt8FewM && few_us < best_us + 3.0 + n * k / 1.4e7) {
        best = Int8Plan{};
        best.few = true;
        best.splits = 1;
    }
    return best;
}

Int8Plan int8_plan(int64_t m, int64_t n, int64_t k, bool tr) {
    if (m <= 0 || n <= 0) return Int8Plan{};
    // a call asks twice (workspace, launch) and a model asks for the same few sizes: the last ones are kept
    struct Kept {
        int64_t m, n, k;
        int cus;
        bool tr;
        Int8Plan p;
    };
    thread_local Kept kept[16] = {};
    const int cus = device_cus();
    Kept& e = kept[(uint64_t)(m * 31 + n * 7 + k) % 16];
    if (e.m != m || e.n != n || e.k != k || e.tr != tr || e.cus != cus)
        e = Kept{m, n, k, cus, tr, make_plan(m, n, k, cus, tr)};
    return e.p;
}

template <int TM, int BN, bool TR, int OUT>
static hipError_t launch_tile(const Int8GemmArgs& a, hipStream_t s) {
    constexpr size_t lds = i8_lds(TM, BN);
    const hipError_t e = allow_dynamic_lds((const void*)int8_gemm_kernel<TM, BN, TR, OUT>, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((int8_gemm_kernel<TM, BN, TR, OUT>), dim3((unsigned)(a.m_tiles * a.n_tiles * a.splits)),
                       dim3(64 * i8_waves(BN)), lds, s, a);
    return hipGetLastError();
}

template <bool TR, int OUT>
static hipError_t launch_way(const Int8GemmArgs& a, int tm, int bn, hipStream_t s) {
    if (bn == 64) return launch_tile<64, 64, TR, OUT>(a, s);
    if (tm == 256) return launch_tile<256, 256, TR, OUT>(a, s);
    if (tm == 128) return launch_tile<128, 256, TR, OUT>(a, s);
    return launch_tile<64, 256, TR, OUT>(a, s);
}

template <int OUT>
static hipError_t launch_out(const Int8GemmArgs& a, const Int8Plan& p, bool tr, hipStream_t s) {
    return tr ? launch_way<true, OUT>(a, p.tm, p.bn, s) : launch_way<false, OUT>(a, p.tm, p.bn, s);
}

template <int MT, int WAVES>
static void launch_few(const Int8GemmArgs& a, int out, unsigned grid, hipStream_t s) {
    const dim3 b(64 * WAVES);
    if (out == DK_FP16)
        hipLaunchKernelGGL((int8_few_kernel<MT, WAVES, DK_FP16>), dim3(grid), b, 0, s, a);
    else if (out == DK_BF16)
        hipLaunchKernelGGL((int8_few_kernel<MT, WAVES, DK_BF16>), dim3(grid), b, 0, s, a);
    else
        hipLaunchKernelGGL((int8_few_kernel<MT, WAVES, DK_FP32>), dim3(grid), b, 0, s, a);
}

template <int DT, int WAVES>
static void launch_few_fused(const Int8GemmArgs& a, const Int8QuantArgs& q, int out, unsigned grid, hipStream_t s) {
    const size_t lds = (size_t)a.m * ((a.k + 63) / 64) * 64;
    const dim3 b(64 * WAVES);
    if (out == DK_FP16)
        hipLaunchKernelGGL((int8_few_fused_kernel<DT, WAVES, DK_FP16>), dim3(grid), b, lds, s, a, q);
    else if (out == DK_BF16)
        hipLaunchKernelGGL((int8_few_fused_kernel<DT, WAVES, DK_BF16>), dim3(grid), b, lds, s, a, q);
    else
        hipLaunchKernelGGL((int8_few_fused_kernel<DT, WAVES, DK_FP32>), dim3(grid), b, lds, s, a, q);
}

bool int8_fused(int64_t m, int64_t k, bool tr) {
    return !tr && m <= kInt8FusedM && m * ((k + 63) / 64) * 64 <= kInt8FusedLds;
}

hipError_t launch_int8_fused(const Int8GemmArgs& a, const Int8QuantArgs& q, int x_dtype, int out_dtype, hipStream_t s) {
    if (a.m == 0 || a.n == 0) return hipSuccess;
    const unsigned grid = (unsigned)((a.n + 15) / 16);
    const bool wide = grid < 512;
    if (x_dtype == DK_FP16)
        wide ? launch_few_fused<DK_FP16, 16>(a, q, out_dtype, grid, s) : launch_few_fused<DK_FP16, 4>(a, q, out_dtype, grid, s);
    else if (x_dtype == DK_BF16)
        wide ? launch_few_fused<DK_BF16, 16>(a, q, out_dtype, grid, s) : launch_few_fused<DK_BF16, 4>(a, q, out_dtype, grid, s);
    else
        wide ? launch_few_fused<DK_FP32, 16>(a, q, out_dtype, grid, s) : launch_few_fused<DK_FP32, 4>(a, q, out_dtype, grid, s);
    return hipGetLastError();
}

hipError_t launch_int8_gemm(Int8GemmArgs a, const Int8Plan& p, int out_dtype, bool tr, hipStream_t s) {
    if (a.m == 0 || a.n == 0) return hipSuccess;
    if (p.few) {
        const unsigned grid = (unsigned)((a.n + 15) / 16);
        // few work-groups with a long k: more waves of each along it ([3584] x 18944 at 8 tokens 27.8 -> 27.0 us;
        // [512] x 3584 is slower with them, 7.8 -> 8.3)
        const bool wide = grid < 512 && a.k >= 8192;
        if (a.m <= 16)
            wide ? launch_few<1, 16>(a, out_dtype, grid, s) : launch_few<1, 4>(a, out_dtype, grid, s);
        else
            wide ? launch_few<2, 16>(a, out_dtype, grid, s) : launch_few<2, 4>(a, out_dtype, grid, s);
        return hipGetLastError();
    }
    a.m_tiles = p.m_tiles;
    a.n_tiles = p.n_tiles;
    a.splits = p.splits;
    a.steps_per_split = p.steps_per_split;
    // an output past the size of the last cache leaves non-temporally ([8192, 18944] 556 -> 543 us); a smaller
    // one stays for its reader, though its own launch would be faster too ([830, 8960] 18.2 against 16.7)
    a.past_caches = a.m * (int64_t)a.n * elem_bytes(out_dtype) > (int64_t(1) << 28);
    if (p.splits == 1) {
        if (out_dtype == DK_FP16) return launch_out<DK_FP16>(a, p, tr, s);
        if (out_dtype == DK_BF16) return launch_out<DK_BF16>(a, p, tr, s);
        return launch_out<DK_FP32>(a, p, tr, s);
    }
    a.ldp = (a.n + 3) / 4 * 4;
    a.slab = (int64_t)a.m * a.ldp;
    const hipError_t e = launch_out<-1>(a, p, tr, s);
    if (e != hipSuccess) return e;
    const unsigned grid = (unsigned)((a.slab / 4 + 255) / 256);
    if (out_dtype == DK_FP16)
        hipLaunchKernelGGL(int8_reduce_kernel<DK_FP16>, dim3(grid), dim3(256), 0, s, a);
    else if (out_dtype == DK_BF16)
        hipLaunchKernelGGL(int8_reduce_kernel<DK_BF16>, dim3(grid), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(int8_reduce_kernel<DK_FP32>, dim3(grid), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace dk
