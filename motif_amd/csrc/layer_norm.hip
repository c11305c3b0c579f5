// Layer normalisation over the last axis, forward and backward.
//
//   forward    m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), y = (x - m) r w + b
//   backward   n = (x - m) r, g = dy w:   dx = r (g - mean(g) - n mean(g n)),   dw = sum over rows of dy n,   db = sum over rows of dy
//
// Bound by memory: forward one read and one write of the data, backward two reads and one write.  A row therefore stays in registers
// between its two reductions (E values in each of L lanes, the mean taken first and the squares of the differences second: no
// cancellation), and the backward pass takes dx and the parameters' sums from the same read: a workgroup walks over rows with its lanes'
// columns fixed, keeps the sums of its columns in registers (fp32) and writes them once; seq_colsum2 adds the workgroups' sums in a fixed
// order.  No atomics: the same bits every time.
// Measured (training): 16384 x 4096 bf16 50 us forward (268 MB, 5.4 TB/s; one workgroup per row and outputs through the caches: 69) and 77 + 5 back
// (403 MB, 5.2 TB/s); 57600 x 64 fp32 8 and 13 + 4; 4099 x 1001 fp16 8 and 15 + 4; 16 x 1024 bf16 3.5, a launch.  Beyond 4096 columns 1024 lanes share a row, with 128 registers
// each: backward no row is requested ahead, and from 8193 columns on the weights, both sums and both inputs of 16 columns do not fit (20 bytes a lane go through scratch in 16 bits,
// 52 in fp32): 4096 x 16384 bf16 65 and 140 (134 MB a tensor, 2.9 TB/s back), fp32 101 and 203.
#include "seq_common.h"

namespace {

constexpr int kMaxD = 16384;                             // 1024 lanes x 16 values

// Sum over the L lanes that share a row, the same value in all of them.  L = 16, 64: lanes of one wave; else the workgroup, through LDS.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* sh) {
    constexpr int W = L < 64 ? L : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (L > 64) {
        __syncthreads();                                 // sh may still be read
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < L / 64; ++i) v += sh[i];
    }
    return v;
}
template <int L>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* sh) {
    constexpr int W = L < 64 ? L : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
    if constexpr (L > 64) {
        constexpr int N = L / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = a; sh[N + (threadIdx.x >> 6)] = b; }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) { a += sh[i]; b += sh[N + i]; }
    }
}

// Run j of a lane: V columns from `c`.  Rows need not be whole runs: the run that would pass the row's end moves back onto the row's last V values,
// and so do those wholly behind it.  What they share with runs before counts for nothing in the sums and is written more than once, alike.
// No access depends on a lane or a row: in a loop whose loads and stores are all taken, the compiler knows how many are younger than the ones
// it waits for, and the wait for the next row's values does not become a wait for this row's stores.
template <int L, int V>
struct Run {
    int c, skip;
    __device__ __forceinline__ Run(int j, int lane, int D) {
        const int first = (j * L + lane) * V;
        c = min(first, D - V);
        skip = first - c;
    }
    __device__ __forceinline__ bool counts(int e) const { return e >= skip; }
};

// A lane's columns of a parameter; `none` where there is no parameter.
template <int L, int V, int NV>
__device__ __forceinline__ void params(const void* p, int D, int pdt, int lane, float none, float (&out)[NV][V]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const Run<L, V> run(j, lane, D);
#pragma unroll
        for (int e = 0; e < V; ++e) out[j][e] = none;
        if (p) seq_param_vec<V>(p, run.c, pdt, out[j]);
    }
}

// A workgroup walks over rows with its columns' weights and biases in registers, the next row requested while this one is summed.
template <typename T, int L, int V, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void layer_norm_fwd_kernel(const T* __restrict__ x, long xs, const void* __restrict__ w, const void* __restrict__ b, int pdt,
                                                                          T* __restrict__ y, float* __restrict__ stats, long rows, int D, float eps, bool stream) {
    __shared__ float sh[32];
    constexpr int TH = L < 256 ? 256 : L, R = TH / L;
    const int lane = threadIdx.x % L;
    const long step = (long)gridDim.x * R;
    SeqRaw<T, V> next[NV];
    auto request = [&](long row) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) next[j] = seq_raw<T, V>(x + row * xs + Run<L, V>(j, lane, D).c);
    };
    const long first = (long)blockIdx.x * R + threadIdx.x / L;
    long row = min(first, rows - 1);                     // (a slot without a row of its own does the last one again)
    request(row);
    float wv[NV][V], bv[NV][V];
    params<L, V, NV>(w, D, pdt, lane, 1.f, wv);
    params<L, V, NV>(b, D, pdt, lane, 0.f, bv);
    for (long base = (long)blockIdx.x * R, at = first; base < rows; base += step) {
        at += step;
        const long next_row = min(at, rows - 1);
        float v[NV][V];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Run<L, V> run(j, lane, D);
#pragma unroll
            for (int e = 0; e < V; ++e) { v[j][e] = next[j][e]; s += run.counts(e) ? v[j][e] : 0.f; }
        }
        request(next_row);
        const float mean = row_sum<L>(s, sh) / (float)D;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Run<L, V> run(j, lane, D);
#pragma unroll
            for (int e = 0; e < V; ++e) { v[j][e] -= mean; q += run.counts(e) ? v[j][e] * v[j][e] : 0.f; }
        }
        const float r = 1.f / sqrtf(row_sum<L>(q, sh) / (float)D + eps);
        if (stats && lane == 0) { stats[2 * row] = mean; stats[2 * row + 1] = r; }
        T* yr = y + row * (long)D;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = v[j][e] * r * wv[j][e] + bv[j][e];
            seq_store<T, V>(yr + Run<L, V>(j, lane, D).c, v[j], stream);
        }
        row = next_row;
    }
}

template <typename T, int L, int V, int NV>
__global__ __launch_bounds__(L < 256 ? 256 : L) void layer_norm_bwd_kernel(const T* __restrict__ x, long xs, const T* __restrict__ dy, long dys, const void* __restrict__ w, int pdt,
                                                                          const float* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, long rows, int D, bool stream) {
    constexpr int TH = L < 256 ? 256 : L, R = TH / L, E = NV * V;
    __shared__ float sh[R > 1 ? 2 * L * E : 64];
    const int lane = threadIdx.x % L, slot = threadIdx.x / L;
    float wv[NV][V], aw[NV][V], ab[NV][V];
    params<L, V, NV>(w, D, pdt, lane, 1.f, wv);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) aw[j][e] = ab[j][e] = 0.f;
    const float inv = 1.f / (float)D;
    typedef SeqRaw<T, V> Raw;
    const long step = (long)gridDim.x * R;
    constexpr bool AHEAD = L < 1024;                     // 16 waves have 128 registers each: none to spare
    Raw xn[NV], dn[NV];                                  // the next row, requested while this one is summed
    float mean_n, r_n;
    auto request = [&](long row) __attribute__((always_inline)) {
        mean_n = stats[2 * row];
        r_n = stats[2 * row + 1];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = Run<L, V>(j, lane, D).c;
            xn[j] = seq_raw<T, V>(x + row * xs + c);
            dn[j] = seq_raw<T, V>(dy + row * dys + c);
        }
    };
    long at = (long)blockIdx.x * R + slot;
    if (AHEAD) request(min(at, rows - 1));
    for (long base = (long)blockIdx.x * R; base < rows; base += step, at += step) {
        const bool on = at < rows;                       // (a slot without a row of its own does the last one again, for no sum)
        const long row = min(at, rows - 1);
        if (!AHEAD) request(row);
        const float mean = mean_n, r = r_n;
        float n[NV][V], g[NV][V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Run<L, V> run(j, lane, D);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                n[j][e] = (xn[j][e] - mean) * r;
                const float d = dn[j][e], gw = d * wv[j][e];
                const bool counts = run.counts(e);       // (in the row's own sums; a row done again counts for no column)
                aw[j][e] += counts && on ? d * n[j][e] : 0.f;
                ab[j][e] += counts && on ? d : 0.f;
                s1 += counts ? gw : 0.f;
                s2 += counts ? gw * n[j][e] : 0.f;
                g[j][e] = gw;
            }
        }
        if (AHEAD) request(min(at + step, rows - 1));
        if (dx) {
            row_sum2<L>(s1, s2, sh);
            s1 *= inv; s2 *= inv;
            T* xo = dx + row * (long)D;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if constexpr (!AHEAD) {                  // (from what was read: n and g of the first walk would not fit)
                    seq_hold(xn[j]);
                    seq_hold(dn[j]);
#pragma unroll
                    for (int e = 0; e < V; ++e) { n[j][e] = (xn[j][e] - mean) * r; g[j][e] = dn[j][e] * wv[j][e]; }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) g[j][e] = r * (g[j][e] - s1 - n[j][e] * s2);
                seq_store<T, V>(xo + Run<L, V>(j, lane, D).c, g[j], stream);
            }
        }
    }
    if (!part) return;
    float* p = part + (long)blockIdx.x * 2 * D;
    if constexpr (R > 1) {                               // the workgroup's R row slots hold the same columns: added in order
        for (int k = 0; k < R; ++k) {
            __syncthreads();
            if (slot == k) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const Run<L, V> run(j, lane, D);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int at = run.c + e;
                        if (!run.counts(e)) continue;
                        sh[at] = k ? sh[at] + aw[j][e] : aw[j][e];
                        sh[L * E + at] = k ? sh[L * E + at] + ab[j][e] : ab[j][e];
                    }
                }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += TH) { p[c] = sh[c]; p[D + c] = sh[L * E + c]; }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const Run<L, V> run(j, lane, D);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (run.counts(e)) { p[run.c + e] = aw[j][e]; p[D + run.c + e] = ab[j][e]; }
        }
    }
}

// 32 columns x 32 row slots per workgroup: a slot adds every 32nd row, the slots are added in order.
__global__ __launch_bounds__(1024) void seq_colsum2_kernel(const float* __restrict__ part, int nb, long D, void* out0, void* out1, int dtype) {
    __shared__ float sh[32][33];
    const int cx = threadIdx.x & 31, slot = threadIdx.x >> 5;
    const long c = (long)blockIdx.x * 32 + cx;
    float s = 0.f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int i = slot; i < nb; i += 32) s += part[(long)i * 2 * D + c];
    }
    sh[slot][cx] = s;
    __syncthreads();
    if (slot == 0 && c < 2 * D) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][cx];
        void* out = c < D ? out0 : out1;
        if (out) seq_param_store(out, c < D ? c : c - D, dtype, t);
    }
}

// The layout of a row: the fewest lanes out of 16 (four rows to a wave), 64 (a wave), 256 and 1024 that hold it with 16 values each, in runs of 16
// bytes; single values for rows shorter than a run.
template <typename T, int L, typename F>
void with_values(int D, F&& f) {
    constexpr int V = 16 / sizeof(T);
    if (D < V) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
    else if (D <= L * V) f(std::integral_constant<int, L>(), std::integral_constant<int, V>(), std::integral_constant<int, 1>());
    else if (D <= L * V * 2) f(std::integral_constant<int, L>(), std::integral_constant<int, V>(), std::integral_constant<int, 2>());
    else f(std::integral_constant<int, L>(), std::integral_constant<int, V>(), std::integral_constant<int, 16 / V>());
}
template <typename T, typename F>
void with_layout(int D, F&& f) {
    if (D <= 16 * 16) with_values<T, 16>(D, f);
    else if (D <= 64 * 16) with_values<T, 64>(D, f);
    else if (D <= 256 * 16) with_values<T, 256>(D, f);
    else with_values<T, 1024>(D, f);
}
// Workgroups: as many as their registers let the chip hold at once, each with a share of the rows (backward: 138 to 146 registers at 16 values of 16 bits a lane, three
// workgroups of 256 to a CU; a fourth share would be a round of its own.  fp32, up to 171, holds two).
int groups_of(long rows, int D, long most) {
    const long want = cdiv(rows, D <= 256 ? 16 : D <= 1024 ? 4 : 1);
    return (int)(want < most ? want : most);
}
int bwd_groups(long rows, int D) { return groups_of(rows, D, D > 4096 ? 512 : D > 512 ? 768 : 1024); }
}  // namespace

int seq_colsum2(const float* part, int nb, long D, void* out0, void* out1, int dtype, hipStream_t s) {
    seq_colsum2_kernel<<<cdiv(2 * D, 32), 1024, 0, s>>>(part, nb, D, out0, out1, dtype);
    MOTIF_LAUNCH_CHECK();
    return MOTIF_OK;
}

extern "C" int motif_layer_norm_fwd(const void* x, long x_rs, const void* weight, const void* bias, void* y, float* stats,
                                    long rows, int D, float eps, int dtype, int param_dtype, void* stream) {
    if (rows < 0 || D < 1 || !seq_dtype_ok(dtype) || !seq_dtype_ok(param_dtype)) return MOTIF_EINVAL;
    if (rows == 0) return MOTIF_OK;
    if (!x || !y || x_rs < 0) return MOTIF_EINVAL;
    if (D > kMaxD || rows > 0x7fffffffL) return MOTIF_ELIMIT;
    seq_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        with_layout<T>(D, [&](auto l, auto v, auto nv) {
            constexpr int L = decltype(l)::value, TH = L < 256 ? 256 : L;
            layer_norm_fwd_kernel<T, L, decltype(v)::value, decltype(nv)::value><<<groups_of(rows, D, 2048), TH, 0, (hipStream_t)stream>>>(
                (const T*)x, x_rs, weight, bias, param_dtype, (T*)y, stats, rows, D, eps, rows * D * (long)sizeof(T) >= kSeqStream);
        });
    });
    MOTIF_LAUNCH_CHECK();
    return MOTIF_OK;
}

extern "C" long motif_layer_norm_bwd_ws_floats(long rows, int D) {
    if (rows < 0 || D < 1) return MOTIF_EINVAL;
    if (D > kMaxD || rows > 0x7fffffffL) return MOTIF_ELIMIT;
    return (long)bwd_groups(rows, D) * 2 * D;
}

extern "C" int motif_layer_norm_bwd(const void* x, long x_rs, const void* dy, long dy_rs, const void* weight, const float* stats, void* dx,
                                    void* dweight, void* dbias, float* workspace, long rows, int D, int dtype, int param_dtype, void* stream) {
    if (rows < 1 || D < 1 || !x || !dy || !stats || x_rs < 0 || dy_rs < 0 || !seq_dtype_ok(dtype) || !seq_dtype_ok(param_dtype)) return MOTIF_EINVAL;
    const bool params = dweight || dbias;
    if ((params && !workspace) || (!params && !dx)) return MOTIF_EINVAL;
    if (D > kMaxD || rows > 0x7fffffffL) return MOTIF_ELIMIT;
    const int nb = bwd_groups(rows, D);
    seq_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        with_layout<T>(D, [&](auto l, auto v, auto nv) {
            constexpr int L = decltype(l)::value, TH = L < 256 ? 256 : L;
            layer_norm_bwd_kernel<T, L, decltype(v)::value, decltype(nv)::value><<<nb, TH, 0, (hipStream_t)stream>>>(
                (const T*)x, x_rs, (const T*)dy, dy_rs, weight, param_dtype, stats, (T*)dx, params ? workspace : nullptr, rows, D, rows * D * (long)sizeof(T) >= kSeqStream);
        });
    });
    MOTIF_LAUNCH_CHECK();
    return params ? seq_colsum2(workspace, nb, D, dweight, dbias, param_dtype, (hipStream_t)stream) : MOTIF_OK;
}
