// The residual stream between two blocks of a decoder layer, a row of `width` elements at a time:
//   rx = 1 / sqrt(mean(x^2) + eps),  p = x rx post_weight        (or p = x: no norm after the block)
//   h = residual_scale residual + gate p                         (gate a channel, a token, an element, or 1)
//   rh = 1 / sqrt(mean(h^2) + eps),  y = h rh weight             (or no y: no norm before the next block)
// and back, with u = gy weight, unit = h rh:
//   dh = gh + rh (u - unit mean(u unit)),  dweight = sum gy unit,  dresidual = residual_scale dh
//   dgate = dh p (summed over what the gate is shared by),  dp = dh gate,  v = dp post_weight
//   dpost_weight = sum dp x rx,  dx = rx (v - x rx mean(v x rx))
// in fp32, one rounding at the end: y and the gradients follow from h as it is before h is rounded, formed again
// from x and residual in the backward.
//
// Layout: a work-group a row, eight columns a thread and pass (a 16-byte load of 16-bit rows), so that the
// row stays in registers between the reductions and is read once; V passes where a row is longer than 512 threads
// take. Work-groups serve rows in turn: the weights and the sums of their gradients stay in
// registers, and the next row's loads fly during the arithmetic of one. A reduction is one barrier: sums of waves go
// to one of two LDS slots in turn, and a slot is written again only after the other's barrier. The sums of
// the weights' gradients leave as a slab a work-group, added in work-group order by a second launch: no atomics, the
// same bits every run.
//
// Bound: HBM at many rows. 8192 x 3584, bf16, both norms and a channel's gate: forward 40.7 us (235 MB, 5.8 TB/s; a large
// copy reaches 5.2), backward 73 (352 MB, 4.8 TB/s) and 4.7 for the join of the slabs; first forms 49 and 119. What took them
// there: waits by count past the stores (every load and store unconditional), weights held in registers, FULL without the
// optional parts' tests, DPP sums and one barrier a reduction, float8 arithmetic without conversions in between.
// Against it: two passes of 256 threads 45.0 and 75.9; twice as many work-groups in the backward 74.9 and 8.4 for the
// join. 830 x 1536, fp16 with an fp32 stream, 6 + 10 + 4 us, 16 rows of 3584 3.7: launches and memory round trips. Rows past
// 8192 columns are read without the next one in flight: 2048 x 16384 back 189 us, 2.4 times its bytes' time.
#include "elem.h"

namespace dk {

constexpr int kNormMaxThreads = 512;  // eight waves: group_sum

// How a row's columns fall to the threads. EVEN: a multiple of eight. TAIL: the last thread takes the last eight columns.
// In both, columns that another thread has as well -- the threads past the row's end repeat its last eight -- are
// computed and written alike (the same values) and left out of the sums: no load or store depends on the thread, so
// that a row's loads are waited for by count, past the stores behind them. SHORT: fewer than eight columns, one thread
// reads them one by one.
enum { EVEN, TAIL, SHORT };

template <int DT, int MODE>
__device__ __forceinline__ typename Elem<DT>::vec fetch8(const typename Elem<DT>::type* p, int n) {
    if constexpr (MODE != SHORT) return load8_raw<DT>(p);
    typename Elem<DT>::vec v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) v[e] = p[e];
    return v;
}

// eight values of a type known at run time
template <int MODE>
__device__ __forceinline__ float8_t fetch8_any(const void* p, int dtype, int64_t at, int n) {
    if (dtype == DK_FP32) return fetch8<DK_FP32, MODE>((const float*)p + at, n);
    if (dtype == DK_BF16) return widen8<DK_BF16>(fetch8<DK_BF16, MODE>((const __bf16*)p + at, n));
    return widen8<DK_FP16>(fetch8<DK_FP16, MODE>((const _Float16*)p + at, n));
}

template <int DT, int MODE>
__device__ __forceinline__ void put8(typename Elem<DT>::type* p, float8_t v, int n) {
    if constexpr (MODE != SHORT) {
        store8<DT>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) store1<DT>(p + e, v[e]);
    }
}

template <int MODE>
__device__ __forceinline__ void put8_any(void* p, int dtype, int64_t at, float8_t v, int n) {
    if (dtype == DK_FP32)
        put8<DK_FP32, MODE>((float*)p + at, v, n);
    else if (dtype == DK_BF16)
        put8<DK_BF16, MODE>((__bf16*)p + at, v, n);
    else
        put8<DK_FP16, MODE>((_Float16*)p + at, v, n);
}

__device__ __forceinline__ float sum8(float8_t v) {
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// v of the lane that a data-parallel primitive names
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// sum over each eight lanes (all get it)
__device__ __forceinline__ float sum_of8(float v) {
    v += dpp<0xB1>(v);          // lanes 1 0 3 2
    v += dpp<0x4E>(v);          // lanes 2 3 0 1
    return v + dpp<0x141>(v);   // mirrored eight
}

// sum over the 64 lanes (all get it) without a round through LDS
__device__ __forceinline__ float wave_sum(float v) {
    v = sum_of8(v);
    v += dpp<0x140>(v);  // mirrored sixteen
    const int u = __builtin_bit_cast(int, v);
    const auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(u, lane)); };
    return (row(0) + row(16)) + (row(32) + row(48));
}

// sums of two values over the work-group (all get them)
__device__ __forceinline__ float2_t group_sum(float a, float b, float2_t* slot) {
    a = wave_sum(a);
    b = wave_sum(b);
    const int waves = blockDim.x / kWave;
    if (waves == 1) return float2_t{a, b};
    if (threadIdx.x % kWave == 0) slot[threadIdx.x / kWave] = float2_t{a, b};
    __syncthreads();
    // the waves' sums, one a lane of each eight, added across the eight
    const int w = threadIdx.x % 8;
    float2_t s = slot[w];
    s = w < waves ? s : float2_t{0.0f, 0.0f};
    return float2_t{sum_of8(s.x), sum_of8(s.y)};
}

// FULL: stream, weight, h (backward: its gradient, and the residual's) are all there, and no row's gate
template <int XT, int ST, int YT, int V, int MODE, bool FULL, bool BWD>
__global__ __launch_bounds__(kNormMaxThreads, V > 1 ? 2 : ST == YT && ST == DK_FP32 ? 3 : 4) void residual_norm_kernel(
    const ResidualNormArgs a) {
#pragma clang fp contract(fast)
    typedef typename Elem<XT>::type x_t;
    typedef typename Elem<ST>::type s_t;
    typedef typename Elem<YT>::type y_t;
    __shared__ float2_t slots[2][kNormMaxThreads / kWave];
    int turn = 0;
    const auto reduce = [&](float p, float q) {
        turn ^= 1;
        return group_sum(p, q, slots[turn]);
    };
    const int width = a.width;
    // this thread's columns of pass v: col[v] .. col[v] + 7, the first skip[v] of them another thread's too
    int col[V], skip[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = 8 * (int)(threadIdx.x + v * blockDim.x);
        col[v] = MODE == SHORT ? 0 : min(c, width - 8);
        skip[v] = MODE == SHORT ? c : min(c - col[v], 8);
    }
    const bool lead = MODE != SHORT || threadIdx.x == 0;
    const int n = MODE == SHORT ? width : 8;
    // the sum over a pass's columns
    const auto sum = [&](float8_t f, int v) {
        if constexpr (MODE == TAIL) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = e < skip[v] ? 0.0f : f[e];
            return sum8(f);
        }
        return skip[v] > 0 ? 0.0f : sum8(f);
    };
    const bool norm = FULL || a.w != nullptr, post = a.pw != nullptr, stream = FULL || a.res != nullptr;
    const bool grad_h = BWD && (FULL || a.gh != nullptr);

    // The weights stay in registers (HOLD), or, four passes, come from the caches at each use. A channel's gate is held as
    // its product with post_weight, and one sum, of dh ux, gives both their gradients in the second launch.
    constexpr bool HOLD = V < 4;
    const bool by_row = !FULL && a.gate_kind > DK_GATE_CHANNEL;
    float8_t held_w[V], held_pw[V], gate_row[V], dw[V], dq[V];
    const auto weight_at = [&](int v) {
        return norm ? fetch8_any<MODE>(a.w, a.w_dtype, col[v], n) : float8_t{};
    };
    const auto branch_weight_at = [&](int v) {
        float8_t q = float8_t{} + 1.0f;
        if (post) q = fetch8_any<MODE>(a.pw, a.pw_dtype, col[v], n);
        if (a.gate_kind == DK_GATE_CHANNEL) q = q * fetch8_any<MODE>(a.gate, a.gate_dtype, col[v], n);
        return q;
    };
    const auto gate_at = [&](int64_t row, int v) -> float8_t {
        if (a.gate_kind == DK_GATE_ELEMENT)
            return fetch8_any<MODE>(a.gate, a.gate_dtype, row * a.ldgate + col[v], n);
        return float8_t{} + load_any(a.gate, a.gate_dtype, row * a.ldgate);
    };
    const auto weight = [&](int v) { return HOLD ? held_w[v] : weight_at(v); };
    const auto branch_weight = [&](int v) { return HOLD ? held_pw[v] : branch_weight_at(v); };
    const auto gate = [&](int64_t row, int v) { return HOLD ? gate_row[v] : gate_at(row, v); };
#pragma unroll
    for (int v = 0; v < V; ++v) {
        dw[v] = dq[v] = float8_t{};
        if constexpr (HOLD) {
            held_w[v] = weight_at(v);
            held_pw[v] = branch_weight_at(v);
        }
    }

    typename Elem<XT>::vec rx8[V];
    typename Elem<ST>::vec rr8[V], rg8[V];
    typename Elem<YT>::vec ry8[V];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rx8[v] = fetch8<XT, MODE>((const x_t*)a.x + row * a.ldx + col[v], n);
            rr8[v] = {};
            if (stream) rr8[v] = fetch8<ST, MODE>((const s_t*)a.res + row * a.ldr + col[v], n);
            if constexpr (BWD) {
                rg8[v] = {};
                ry8[v] = {};
                if (grad_h) rg8[v] = fetch8<ST, MODE>((const s_t*)a.gh + row * a.ldgh + col[v], n);
                if (norm) ry8[v] = fetch8<YT, MODE>((const y_t*)a.gy + row * a.ldgy + col[v], n);
            }
        }
    };

    int row = blockIdx.x;
    if (HOLD) fetch(min(row, a.rows - 1));
    for (; row < a.rows; row += gridDim.x) {
        float8_t x[V], h[V], gh[V], gy[V];
        const int64_t at = (int64_t)row * width;
        if constexpr (!HOLD) fetch(row);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = widen8<XT>(rx8[v]);
            h[v] = widen8<ST>(rr8[v]) * a.scale;  // zeros without a stream
            if (!FULL && !stream) h[v] = float8_t{};
            if constexpr (BWD) {
                gh[v] = widen8<ST>(rg8[v]);
                gy[v] = widen8<YT>(ry8[v]);
            }
            if (HOLD && by_row) gate_row[v] = gate_at(row, v);
        }
        if constexpr (HOLD) {
            // the loaded registers are free for the next row: without this they live on, and copies of the next row's
            // wait for its loads at the end of this one
#pragma unroll
            for (int v = 0; v < V; ++v) {
                asm volatile("" : "+v"(x[v]), "+v"(h[v]));
                if constexpr (BWD) asm volatile("" : "+v"(gh[v]), "+v"(gy[v]));
            }
            fetch(min(row + (int)gridDim.x, a.rows - 1));
        }

        float rx = 1.0f;
        if (post) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) s += sum(x[v] * x[v], v);
            rx = rsqrtf(reduce(s, 0.0f).x * a.inv_width + a.eps);
        }
        // x becomes the normalized row
        float sh = 0.0f, su = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = x[v] * rx;
            const float8_t p = x[v] * branch_weight(v);
            h[v] = h[v] + (by_row ? gate(row, v) * p : p);
            sh += sum(h[v] * h[v], v);
            if constexpr (BWD) {
                if (norm) su += sum(gy[v] * weight(v) * h[v], v);
            }
        }
        if constexpr (!BWD) {
            if (FULL || a.h != nullptr) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (lead) put8<ST, MODE>((s_t*)a.h + at + col[v], h[v], n);
            }
            if (norm) {
                const float rh = rsqrtf(reduce(sh, 0.0f).x * a.inv_width + a.eps);
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (lead) put8<YT, MODE>((y_t*)a.y + at + col[v], h[v] * rh * weight(v), n);
            }
        } else {
            if (norm) {
                const float2_t s = reduce(sh, su);
                const float rh = rsqrtf(s.x * a.inv_width + a.eps);
                const float mean = s.y * rh * a.inv_width;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float8_t unit = h[v] * rh;
                    dw[v] = dw[v] + gy[v] * unit;
                    gh[v] = gh[v] + (gy[v] * weight(v) - unit * mean) * rh;
                }
            }
            // gh is dh from here on
            float sv = 0.0f, sg = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if ((FULL || a.dres != nullptr) && lead) put8<ST, MODE>((s_t*)a.dres + at + col[v], gh[v] * a.scale, n);
                if (by_row) {
                    const float8_t dg = gh[v] * (x[v] * branch_weight(v));
                    if (a.gate_kind == DK_GATE_TOKEN)
                        sg += sum(dg, v);
                    else if (a.dgate != nullptr && lead)
                        put8_any<MODE>(a.dgate, a.gate_dtype, at + col[v], dg, n);
                    gh[v] = gh[v] * gate(row, v);
                }
                dq[v] = dq[v] + gh[v] * x[v];
                gh[v] = gh[v] * branch_weight(v);
                if (post) sv += sum(gh[v] * x[v], v);
            }
            if (post || (!FULL && a.gate_kind == DK_GATE_TOKEN)) {
                const float2_t s = reduce(sv, sg);
                if (!FULL && a.gate_kind == DK_GATE_TOKEN && a.dgate != nullptr && threadIdx.x == 0) {
                    if (a.gate_dtype == DK_FP32)
                        store1<DK_FP32>((float*)a.dgate + row, s.y);
                    else if (a.gate_dtype == DK_BF16)
                        store1<DK_BF16>((__bf16*)a.dgate + row, s.y);
                    else
                        store1<DK_FP16>((_Float16*)a.dgate + row, s.y);
                }
                if (post) {
                    const float mean = s.x * a.inv_width;
#pragma unroll
                    for (int v = 0; v < V; ++v) gh[v] = (gh[v] - x[v] * mean) * rx;
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (lead) put8<XT, MODE>((x_t*)a.dx + at + col[v], gh[v], n);
        }
    }
    if constexpr (BWD) {
        if (a.slabs == nullptr) return;
        float* slab = a.slabs + (int64_t)blockIdx.x * a.nslabs * width;
        const auto leave = [&](const float8_t* sums) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (lead) put8<DK_FP32, MODE>(slab + col[v], sums[v], n);
            slab += width;
        };
        if (a.slab_w) leave(dw);
        if (a.slab_q) leave(dq);
    }
}

// Columns of all slabs (dweight's sums, then those of dh ux), each added by 16 threads in slab order, then those in a
// fixed order.
constexpr int kSumCols = 64, kSumRows = 16;
__global__ __launch_bounds__(kSumCols* kSumRows) void residual_norm_sum_kernel(const ResidualNormArgs a, int n, float* dw,
                                                                               float* dpw, float* dgate) {
    __shared__ float part[kSumRows][kSumCols];
    const int cx = threadIdx.x % kSumCols, ry = threadIdx.x / kSumCols;
    const int cols = a.nslabs * a.width, col = blockIdx.x * kSumCols + cx;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (int i = ry; i < n; i += kSumRows) v += a.slabs[(int64_t)i * cols + col];
    }
    part[ry][cx] = v;
    __syncthreads();
    if (ry == 0 && col < cols) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kSumRows; ++i) s += part[i][cx];
        if (a.slab_w && col < a.width) {
            dw[col] = s;
        } else {
            const int c = a.slab_w ? col - a.width : col;
            if (dpw != nullptr) dpw[c] = a.gate_kind == DK_GATE_CHANNEL ? s * load_any(a.gate, a.gate_dtype, c) : s;
            if (dgate != nullptr) dgate[c] = a.pw != nullptr ? s * load_any(a.pw, a.pw_dtype, c) : s;
        }
    }
}

static int norm_passes(int width) { return width <= 8 * kNormMaxThreads ? 1 : width <= 16 * kNormMaxThreads ? 2 : 4; }

static int norm_threads(int width) {
    const int per = 8 * norm_passes(width);
    return ((width + per - 1) / per + kWave - 1) / kWave * kWave;
}

// Work-groups: as many as the CUs hold at once, each with several rows where there are many. In the backward each leaves a
// slab, which costs as much as a third of a row to four fifths: up to four rows a work-group once there are enough for
// the CUs. (us of the backward and its join at one, two, three, four rows: 830 x 1536 fp16 with an fp32 stream 15.1, 12.7, 12.6,
// 13.4; 512 x 3584 13.0, 11.0, 11.4, 11.0; 2048 x 1536 23.1, 21.2, 21.6, 20.1; 128 x 3584 9.6, 10.7, 11.8, 13.1; 333 x 1121
// from memory 12.4, 13.5; and
// 1024 x 8192, of which a CU holds one work-group, 39.5 with two a CU, 31.4 with one.)
int residual_norm_groups(int64_t rows, int width, bool backward) {
    const int waves = norm_threads(width) / kWave;
    if (!backward) {
        const int64_t want = (24 + waves - 1) / waves * 256;
        return (int)(rows < want ? rows : want);
    }
    const int64_t want = (norm_passes(width) > 1 ? 1 : 16 / waves) * 256, each = (rows + 127) / 256;
    const int64_t few = each <= 1 ? rows : (rows + (each < 4 ? each : 4) - 1) / (each < 4 ? each : 4);
    return (int)(few < want ? few : want);
}

template <int XT, int ST, int YT, int V, int MODE, bool BWD>
static void launch_full(const ResidualNormArgs& a, unsigned grid, hipStream_t s) {
    const dim3 g(grid), t(norm_threads(a.width));
    const bool ends = BWD ? a.gh != nullptr && a.dres != nullptr : a.h != nullptr;
    if (V < 4 && ends && a.res != nullptr && a.w != nullptr && a.gate_kind <= DK_GATE_CHANNEL)
        hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, V, MODE, (V < 4), BWD>), g, t, 0, s, a);
    else
        hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, V, MODE, false, BWD>), g, t, 0, s, a);
}

template <int XT, int ST, int YT, bool BWD>
static void launch_sized(const ResidualNormArgs& a, unsigned grid, hipStream_t s) {
    const int passes = norm_passes(a.width);
    if (a.width < 8)
        hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, 1, SHORT, false, BWD>), dim3(grid),
                           dim3(norm_threads(a.width)), 0, s, a);
    else if (a.width % 8 == 0)
        passes == 1   ? launch_full<XT, ST, YT, 1, EVEN, BWD>(a, grid, s)
        : passes == 2 ? launch_full<XT, ST, YT, 2, EVEN, BWD>(a, grid, s)
                      : launch_full<XT, ST, YT, 4, EVEN, BWD>(a, grid, s);
    else
        passes == 1   ? launch_full<XT, ST, YT, 1, TAIL, BWD>(a, grid, s)
        : passes == 2 ? launch_full<XT, ST, YT, 2, TAIL, BWD>(a, grid, s)
                      : launch_full<XT, ST, YT, 4, TAIL, BWD>(a, grid, s);
}

template <bool BWD>
static void launch_typed(const ResidualNormArgs& a, int x, int st, int y, unsigned grid, hipStream_t s) {
    if (x == DK_FP32)
        launch_sized<DK_FP32, DK_FP32, DK_FP32, BWD>(a, grid, s);
    else if (x == DK_FP16) {
        if (st == x && y == x) launch_sized<DK_FP16, DK_FP16, DK_FP16, BWD>(a, grid, s);
        else if (st == x) launch_sized<DK_FP16, DK_FP16, DK_FP32, BWD>(a, grid, s);
        else if (y == x) launch_sized<DK_FP16, DK_FP32, DK_FP16, BWD>(a, grid, s);
        else launch_sized<DK_FP16, DK_FP32, DK_FP32, BWD>(a, grid, s);
    } else {
        if (st == x && y == x) launch_sized<DK_BF16, DK_BF16, DK_BF16, BWD>(a, grid, s);
        else if (st == x) launch_sized<DK_BF16, DK_BF16, DK_FP32, BWD>(a, grid, s);
        else if (y == x) launch_sized<DK_BF16, DK_FP32, DK_BF16, BWD>(a, grid, s);
        else launch_sized<DK_BF16, DK_FP32, DK_FP32, BWD>(a, grid, s);
    }
}

hipError_t launch_residual_norm(ResidualNormArgs a, int x_dtype, int stream_dtype, int y_dtype, bool backward,
                                float* dw, float* dpw, float* dgate_channel, hipStream_t s) {
    const unsigned grid = (unsigned)residual_norm_groups(a.rows, a.width, backward);
    if (a.rows > 0) {
        if (backward)
            launch_typed<true>(a, x_dtype, stream_dtype, y_dtype, grid, s);
        else
            launch_typed<false>(a, x_dtype, stream_dtype, y_dtype, grid, s);
    }
    if (a.nslabs > 0)
        hipLaunchKernelGGL(residual_norm_sum_kernel, dim3((a.nslabs * a.width + kSumCols - 1) / kSumCols),
                           dim3(kSumCols * kSumRows), 0, s, a, (int)grid, dw, dpw, dgate_channel);
    return hipGetLastError();
}

}  // namespace dk
