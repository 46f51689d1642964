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
#include "elem.h"

namespace dk {

constexpr int kNormMaxThreads = 512;

template <int DT>
__device__ __forceinline__ typename Elem<DT>::vec fetch8(const typename Elem<DT>::type* p, int n) {
    if (n >= 8) return load8_raw<DT>(p);
    typename Elem<DT>::vec v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) v[e] = p[e];
    return v;
}

// eight values of a type known at run time; n of them exist
__device__ __forceinline__ float8_t fetch8_any(const void* p, int dtype, int64_t at, int n) {
    if (dtype == DK_FP32) return fetch8<DK_FP32>((const float*)p + at, n);
    if (dtype == DK_BF16) return widen8<DK_BF16>(fetch8<DK_BF16>((const __bf16*)p + at, n));
    return widen8<DK_FP16>(fetch8<DK_FP16>((const _Float16*)p + at, n));
}

template <int DT>
__device__ __forceinline__ void put8(typename Elem<DT>::type* p, float8_t v, int n) {
    if (n >= 8) {
        store8<DT>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) store1<DT>(p + e, v[e]);
    }
}

__device__ __forceinline__ void put8_any(void* p, int dtype, int64_t at, float8_t v, int n) {
    if (dtype == DK_FP32)
        put8<DK_FP32>((float*)p + at, v, n);
    else if (dtype == DK_BF16)
        put8<DK_BF16>((__bf16*)p + at, v, n);
    else
        put8<DK_FP16>((_Float16*)p + at, v, n);
}

__device__ __forceinline__ float sum8(float8_t v) {
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// sums of two values over the work-group (all get them)
__device__ __forceinline__ float2_t group_sum(float a, float b, float2_t* slot) {
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    const int waves = blockDim.x / kWave;
    if (waves == 1) return float2_t{a, b};
    if (threadIdx.x % kWave == 0) slot[threadIdx.x / kWave] = float2_t{a, b};
    __syncthreads();
    float2_t s = slot[0];
    for (int w = 1; w < waves; ++w) {
        const float2_t o = slot[w];
        s.x += o.x;
        s.y += o.y;
    }
    return s;
}

template <int XT, int ST, int YT, int V, bool BWD>
__global__ __launch_bounds__(kNormMaxThreads) void residual_norm_kernel(const ResidualNormArgs a) {
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
    int col[V], n[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = 8 * (int)(threadIdx.x + v * blockDim.x);
        n[v] = min(max(width - col[v], 0), 8);
        if (n[v] == 0) col[v] = 0;
    }
    const bool norm = a.w != nullptr, post = a.pw != nullptr, stream = a.res != nullptr;
    const bool grad_h = BWD && a.gh != nullptr;

    // weights and gate stay in registers (HOLD), or, four passes, come from the caches at each use
    constexpr bool HOLD = V < 4;
    float8_t held_w[V], held_pw[V], held_gate[V], dw[V], dpw[V], dgate[V];
    const auto gate_at = [&](int64_t row, int v) -> float8_t {
        if (a.gate_kind == DK_GATE_CHANNEL) return fetch8_any(a.gate, a.gate_dtype, col[v], n[v]);
        if (a.gate_kind == DK_GATE_ELEMENT) return fetch8_any(a.gate, a.gate_dtype, row * a.ldgate + col[v], n[v]);
        if (a.gate_kind == DK_GATE_TOKEN) return float8_t{} + load_any(a.gate, a.gate_dtype, row * a.ldgate);
        return float8_t{} + 1.0f;
    };
    const auto weight = [&](int v) { return HOLD ? held_w[v] : fetch8_any(a.w, a.w_dtype, col[v], n[v]); };
    const auto post_weight = [&](int v) { return HOLD ? held_pw[v] : fetch8_any(a.pw, a.pw_dtype, col[v], n[v]); };
    const auto gate = [&](int64_t row, int v) { return HOLD ? held_gate[v] : gate_at(row, v); };
#pragma unroll
    for (int v = 0; v < V; ++v) {
        dw[v] = dpw[v] = dgate[v] = float8_t{};
        if constexpr (HOLD) {
            held_w[v] = norm ? fetch8_any(a.w, a.w_dtype, col[v], n[v]) : float8_t{};
            held_pw[v] = post ? fetch8_any(a.pw, a.pw_dtype, col[v], n[v]) : float8_t{};
            if (a.gate_kind <= DK_GATE_CHANNEL) held_gate[v] = gate_at(0, v);
        }
    }

    typename Elem<XT>::vec rx8[V];
    typename Elem<ST>::vec rr8[V], rg8[V];
    typename Elem<YT>::vec ry8[V];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rx8[v] = fetch8<XT>((const x_t*)a.x + row * a.ldx + col[v], n[v]);
            if (stream) rr8[v] = fetch8<ST>((const s_t*)a.res + row * a.ldr + col[v], n[v]);
            if constexpr (BWD) {
                if (grad_h) rg8[v] = fetch8<ST>((const s_t*)a.gh + row * a.ldgh + col[v], n[v]);
                if (norm) ry8[v] = fetch8<YT>((const y_t*)a.gy + row * a.ldgy + col[v], n[v]);
            }
        }
    };

    int row = blockIdx.x;
    if (HOLD && row < a.rows) fetch(row);
    for (; row < a.rows; row += gridDim.x) {
        float8_t x[V], h[V], gh[V], gy[V];
        const int64_t at = (int64_t)row * width;
        if constexpr (!HOLD) fetch(row);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = widen8<XT>(rx8[v]);
            h[v] = stream ? widen8<ST>(rr8[v]) * a.scale : float8_t{};
            gh[v] = gy[v] = float8_t{};
            if constexpr (BWD) {
                if (grad_h) gh[v] = widen8<ST>(rg8[v]);
                if (norm) gy[v] = widen8<YT>(ry8[v]);
            }
            if (HOLD && a.gate_kind > DK_GATE_CHANNEL) held_gate[v] = gate_at(row, v);
        }
        if (HOLD && row + (int)gridDim.x < a.rows) fetch(row + gridDim.x);

        float rx = 1.0f;
        if (post) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) s += sum8(x[v] * x[v]);
            rx = rsqrtf(reduce(s, 0.0f).x * a.inv_width + a.eps);
        }
        // x becomes the normalized row, branch() what the gate takes
        const auto branch = [&](int v) { return post ? x[v] * post_weight(v) : x[v]; };
        float sh = 0.0f, su = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = x[v] * rx;
            h[v] = h[v] + gate(row, v) * branch(v);
            sh += sum8(h[v] * h[v]);
            if constexpr (BWD) {
                if (norm) su += sum8(gy[v] * weight(v) * h[v]);
            }
        }
        if constexpr (!BWD) {
            if (a.h != nullptr) {
#pragma unroll
                for (int v = 0; v < V; ++v) put8<ST>((s_t*)a.h + at + col[v], h[v], n[v]);
            }
            if (norm) {
                const float rh = rsqrtf(reduce(sh, 0.0f).x * a.inv_width + a.eps);
#pragma unroll
                for (int v = 0; v < V; ++v) put8<YT>((y_t*)a.y + at + col[v], h[v] * rh * weight(v), n[v]);
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
                if (a.dres != nullptr) put8<ST>((s_t*)a.dres + at + col[v], gh[v] * a.scale, n[v]);
                const float8_t dg = gh[v] * branch(v);
                if (a.gate_kind == DK_GATE_CHANNEL)
                    dgate[v] = dgate[v] + dg;
                else if (a.gate_kind == DK_GATE_ELEMENT && a.dgate != nullptr)
                    put8_any(a.dgate, a.gate_dtype, at + col[v], dg, n[v]);
                sg += sum8(dg);
                gh[v] = gh[v] * gate(row, v);
                if (post) {
                    dpw[v] = dpw[v] + gh[v] * x[v];
                    gh[v] = gh[v] * post_weight(v);
                    sv += sum8(gh[v] * x[v]);
                }
            }
            if (post || a.gate_kind == DK_GATE_TOKEN) {
                const float2_t s = reduce(sv, sg);
                if (a.gate_kind == DK_GATE_TOKEN && a.dgate != nullptr && threadIdx.x == 0) {
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
            for (int v = 0; v < V; ++v) put8<XT>((x_t*)a.dx + at + col[v], gh[v], n[v]);
        }
    }
    if constexpr (BWD) {
        if (a.slabs == nullptr) return;
        float* slab = a.slabs + (int64_t)blockIdx.x * a.nslabs * width;
        const auto leave = [&](const float8_t* sums) {
#pragma unroll
            for (int v = 0; v < V; ++v) put8<DK_FP32>(slab + col[v], sums[v], n[v]);
            slab += width;
        };
        if (a.slab_w) leave(dw);
        if (a.slab_pw) leave(dpw);
        if (a.slab_gate) leave(dgate);
    }
}

// columns of all slabs, `cols` a slab: each added by 16 threads in slab order, then those in a fixed order
constexpr int kSumCols = 64, kSumRows = 16;
__global__ __launch_bounds__(kSumCols* kSumRows) void slab_sum_kernel(const float* __restrict__ slabs, int n, int cols,
                                                                      int width, float* o0, float* o1, float* o2) {
    __shared__ float part[kSumRows][kSumCols];
    const int cx = threadIdx.x % kSumCols, ry = threadIdx.x / kSumCols;
    const int col = blockIdx.x * kSumCols + cx;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (int i = ry; i < n; i += kSumRows) v += slabs[(int64_t)i * cols + col];
    }
    part[ry][cx] = v;
    __syncthreads();
    if (ry == 0 && col < cols) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kSumRows; ++i) s += part[i][cx];
        const int which = col / width;
        (which == 0 ? o0 : which == 1 ? o1 : o2)[col - which * width] = s;
    }
}

static int norm_passes(int width) { return width <= 8 * kNormMaxThreads ? 1 : width <= 16 * kNormMaxThreads ? 2 : 4; }

static int norm_threads(int width) {
    const int per = 8 * norm_passes(width);
    return ((width + per - 1) / per + kWave - 1) / kWave * kWave;
}

// Work-groups: as many as the CUs hold at once, each with several rows where there are many.
int residual_norm_groups(int64_t rows, int width, bool backward) {
    const int waves = norm_threads(width) / kWave;
    const int64_t per_cu = backward ? (12 + waves - 1) / waves : (24 + waves - 1) / waves;
    const int64_t want = per_cu * 256;
    return (int)(rows < want ? rows : want);
}

template <int XT, int ST, int YT, bool BWD>
static void launch_sized(const ResidualNormArgs& a, unsigned grid, hipStream_t s) {
    const dim3 threads(norm_threads(a.width));
    switch (norm_passes(a.width)) {
        case 1: hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, 1, BWD>), dim3(grid), threads, 0, s, a); break;
        case 2: hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, 2, BWD>), dim3(grid), threads, 0, s, a); break;
        default: hipLaunchKernelGGL((residual_norm_kernel<XT, ST, YT, 4, BWD>), dim3(grid), threads, 0, s, a); break;
    }
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
    if (a.nslabs > 0) {
        float* out[3] = {nullptr, nullptr, nullptr};
        int i = 0;
        if (a.slab_w) out[i++] = dw;
        if (a.slab_pw) out[i++] = dpw;
        if (a.slab_gate) out[i++] = dgate_channel;
        const int cols = a.nslabs * a.width;
        hipLaunchKernelGGL(slab_sum_kernel, dim3((cols + kSumCols - 1) / kSumCols), dim3(kSumCols * kSumRows), 0, s,
                           a.slabs, (int)grid, cols, a.width, out[0], out[1], out[2]);
    }
    return hipGetLastError();
}

}  // namespace dk
