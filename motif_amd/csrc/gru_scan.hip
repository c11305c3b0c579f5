// The recurrence of motif_gru_update over whole sequences, for gates that do not read the state:
//
//   forward    h_t = a_t h_{t-1} + z_t q_t,   a_t = 1 - z_t                         channel by channel
//   backward   g_t = dh_t + c_t,  c_{t-1} = a_t g_t  (c of the last row: the gradient of the last state)
//              dq_t = g_t z_t,    dz_t = g_t (q_t - h_{t-1}),    dh0 = a_0 g_0
//
// Both are first-order linear recurrences; the backward one runs from the end.  A run of rows acts on the state that enters it as
// x -> A x + H, and two runs compose as (A2 A1, A2 H1 + H2): that is what lets time be split.  Sequences packed one behind the other are one recurrence
// over all rows: a run that holds a sequence's first row (or a row of none) is marked as cut and composes as (0, H2) with what lies before it,
// whatever that is -- an infinite state of one sequence must not meet the next one's 0.
//
// Bound by memory (forward 2 reads and 1 write, backward 4 reads and 2 writes of the data).  A workgroup owns TX lanes x V channels and TY time
// slots of R rows each: a tile of TY R rows lies in registers, as it was read, between the composition of its slots (lanes of a wave by shuffles, the waves
// through LDS) and the second walk over its rows that writes them.  TY = 1 where channels alone fill the chip or the sequence is short.  Where
// channels are few, a sequence is cut into segments: a first kernel reads what the composition needs and writes every segment's (A, H), and each
// segment's workgroup then composes those before it, in a fixed order -- the cost is a second read of half the inputs.  The states, A and H are
// fp32.  No atomics: the same bits every time.
// Measured: 65536 x 1024 bf16 51 + 71 us forward (two reads, then two reads and a write: 5.3 and 5.7 TB/s), 43 + 176 back (4.6 TB/s in the second);
// 7 x 3686400 fp32, one lane per four channels, 64 (310 MB, 4.9 TB/s) and 114 back (619 MB, 5.4 TB/s; forward 54 in a row of its own calls); 20011 x 771 fp16 in 37 sequences
// 4 + 22 + 46 and 4 + 22 + 78: three tiles to a workgroup do not hide their first reads.  Where z leaves 0 .. 1 far enough for a run's A to pass fp32's range, the split form gives NaN even
// where the state itself stays finite.
#include "seq_common.h"

namespace {

struct ScanArgs {
    const void *z, *q, *h, *dh;                          // q, h: backward's second kernel and forward; dh: backward
    const float *h0, *dlast;
    void *out0, *out1;                                   // forward: h, -; backward: dz, dq (either may be null)
    float* state;                                        // forward: the last states, backward: dh0 (may be null)
    float* agg;                                          // [B][segs][2][D], null with one segment
    int* cuts;                                           // packed: whether a segment is cut, [segs]
    const int* info;                                     // packed rows: owner << 2 | last << 1 | first, -1: no sequence's row.  null: B sequences of T rows
    long zb, zr, qb, qr, db, dr;                         // batch and row strides of z, q, dh; h, out0 and out1 are dense
    long T, seg_rows;
    int B, D, groups, segs;                              // groups: workgroups that share a batch's channels, TY = 1: lanes
    bool stream;
};

constexpr int kFirst = 1, kLast = 2;

template <int V, int TX, int TY>
struct Slots {                                           // 256 threads: TX lanes across channels, TY time slots
    static constexpr int WX = TX < 64 ? TX : 64, WY = 64 / WX, WAVES = TY > 1 ? 4 : 1;
    static_assert(TX * TY == 256 && (TY == 1 || TX <= 64), "");

    struct Sums { float v[4][2][TX * V]; int cut[4]; };  // of the waves

    // A, H (and the cut) of this slot -> of the slots in front of it in its wave; the wave's own to sums
    template <bool PACKED>
    static __device__ __forceinline__ void wave_scan(float (&A)[V], float (&H)[V], int& cut, Sums& sums) {
        const int lane = threadIdx.x & 63, sy = lane / WX, tx = lane % WX, wave = threadIdx.x >> 6;
#pragma unroll
        for (int d = 1; d < WY; d <<= 1) {
            const int oc = PACKED ? __shfl_up(cut, d * WX) : 0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float oa = __shfl_up(A[v], d * WX), oh = __shfl_up(H[v], d * WX);
                if (sy >= d && !(PACKED && cut)) { H[v] = fmaf(A[v], oh, H[v]); A[v] *= oa; }
            }
            if (PACKED && sy >= d) cut |= oc;
        }
        if (sy == WY - 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) { sums.v[wave][0][tx * V + v] = A[v]; sums.v[wave][1][tx * V + v] = H[v]; }
            if (PACKED && tx == 0) sums.cut[wave] = cut; // (the same in every lane of a slot that has channels; the first always has)
        }
        const int oc = PACKED && WY > 1 ? __shfl_up(cut, WX) : 0;
        if (PACKED) cut = sy ? oc : 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float oa = WY > 1 ? __shfl_up(A[v], WX) : 1.f, oh = WY > 1 ? __shfl_up(H[v], WX) : 0.f;
            A[v] = sy ? oa : 1.f;
            H[v] = sy ? oh : 0.f;
        }
    }
    // behind a barrier: the state that enters this wave's slots, and `carry` moved past all waves
    template <bool PACKED>
    static __device__ __forceinline__ void waves_apply(float (&carry)[V], float (&in)[V], const Sums& sums, int tx) {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const bool cut = PACKED && sums.cut[w];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (w == wave) in[v] = carry[v];
                carry[v] = cut ? sums.v[w][1][tx * V + v] : fmaf(sums.v[w][0][tx * V + v], carry[v], sums.v[w][1][tx * V + v]);
            }
        }
    }
};

template <int V>
__device__ __forceinline__ void zero(float (&x)[V], float c = 0.f) {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = c;
}

// One row more behind a run: forward  x -> a x + z q,   backward  c -> a (c + dh).  Packed: a sequence's first row in the recurrence's order starts
// from the sequence's own state, a row of none from nothing; both cut.
template <bool BWD, bool PACKED, int V, typename X>
__device__ __forceinline__ void compose(float (&A)[V], float (&H)[V], int& cut, const X& z, const X& x, int flag, const float* init, int c0, int D) {
    if (PACKED && (flag < 0 || (flag & (BWD ? kLast : kFirst)))) {
        cut = 1;
        zero(A);
        zero(H);
        if (flag >= 0 && init) seq_load<float, V>(init + (long)(flag >> 2) * D + c0, H);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float a = 1.f - z[v], n = BWD ? a * (H[v] + x[v]) : fmaf(a, H[v], z[v] * x[v]);
        H[v] = PACKED && flag < 0 ? 0.f : n;
        A[v] = PACKED && flag < 0 ? 0.f : A[v] * a;
    }
}

struct Where { int group, seg; long b; };
__device__ __forceinline__ Where where(const ScanArgs& p) {
    const long bs = blockIdx.x / p.groups;
    return {(int)(blockIdx.x % p.groups), (int)(bs % p.segs), bs / p.segs};
}

// (A, H) of every segment but the last: each slot walks its own run of the segment's rows, four rows at a time, the next four requested ahead.
template <typename T, int V, int TX, int TY, bool BWD, bool PACKED>
__global__ __launch_bounds__(256) void gru_scan_segments_kernel(ScanArgs p) {
    using S = Slots<V, TX, TY>;
    __shared__ typename S::Sums sums;
    const Where at = where(p);
    if (at.seg == p.segs - 1) return;
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, first = (at.group * TX + tx) * V, c0 = min(first, p.D - V);
    const bool on = first < p.D;                         // (the last lanes of a row take its last V channels: those they share are written more than once, alike)
    const T* z = (const T*)p.z + at.b * p.zb + c0;
    const T* x = BWD ? (const T*)p.dh + at.b * p.db + c0 : (const T*)p.q + at.b * p.qb + c0;
    const long xr = BWD ? p.dr : p.qr;
    const long run = p.seg_rows / TY, k0 = at.seg * p.seg_rows + ty * run;     // rows in the order of the recurrence; a segment that is not the last is full
    struct Rows { SeqRaw<T, V> z[4], x[4]; int f[4]; };
    auto read = [&](Rows& w, long k) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long t = BWD ? p.T - 1 - (k + r) : k + r;
            w.z[r] = seq_raw<T, V>(z + t * p.zr);
            w.x[r] = seq_raw<T, V>(x + t * xr);
            if (PACKED) w.f[r] = p.info[t];
        }
    };
    float A[V], H[V];
    int cut = 0;
    zero(A, 1.f);
    zero(H);
    {
        Rows now, next;
        read(now, k0);
        for (long k = k0; k < k0 + run; k += 4) {
            read(next, min(k + 4, k0 + run - 4));        // (always taken: the compiler counts the requests behind the one it waits for)
#pragma unroll
            for (int r = 0; r < 4; ++r) compose<BWD, PACKED, V>(A, H, cut, now.z[r], now.x[r], now.f[r], BWD ? p.dlast : p.h0, c0, p.D);
            now = next;
        }
    }
    S::template wave_scan<PACKED>(A, H, cut, sums);
    __syncthreads();
    if (ty == 0 && on) {
        float* o = p.agg + ((at.b * p.segs + at.seg) * 2) * p.D + c0;
        zero(A, 1.f);
        zero(H);
        cut = 0;
#pragma unroll
        for (int w = 0; w < S::WAVES; ++w) {
            const bool c = PACKED && sums.cut[w];
            cut |= c;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                H[v] = c ? sums.v[w][1][tx * V + v] : fmaf(sums.v[w][0][tx * V + v], H[v], sums.v[w][1][tx * V + v]);
                A[v] = c ? 0.f : sums.v[w][0][tx * V + v] * A[v];
            }
        }
        seq_store<float, V>(o, A);
        seq_store<float, V>(o + p.D, H);
        if (PACKED && first == 0) p.cuts[at.seg] = cut;
    }
}

template <typename T, int V, int TX, int TY, int R, bool BWD, bool PACKED>
__global__ __launch_bounds__(256) void gru_scan_kernel(ScanArgs p) {
    using S = Slots<V, TX, TY>;
    __shared__ typename S::Sums sums[2];
    // TY = 1: the lanes of all batches one behind the other, `groups` to a batch (host: below 2^32 in all; those behind the last do its work again, and write alike)
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const unsigned n = min(blockIdx.x * 256u + threadIdx.x, (unsigned)p.B * (unsigned)p.groups - 1u);
    const Where at = TY == 1 ? Where{(int)(n % (unsigned)p.groups), 0, (long)(n / (unsigned)p.groups)} : where(p);
    const int c0 = min((TY == 1 ? at.group : at.group * TX + tx) * V, p.D - V);      // (the last lanes of a row take its last V channels: those they share are written more than once, alike)
    // Addresses: a uniform row of the tile, and a lane's offset from it in bytes (32 bits: the host bounds the strides where TY > 1).  Backward, time
    // runs down: slot TY - 1 has the tile's first rows.
    const int slot = (BWD ? TY - 1 - ty : ty) * R;
    const unsigned oz = (unsigned)(slot * (unsigned)p.zr + c0) * sizeof(T), oq = (unsigned)(slot * (unsigned)p.qr + c0) * sizeof(T);
    const unsigned od = BWD ? (unsigned)(slot * (unsigned)p.dr + c0) * sizeof(T) : 0u, oo = (unsigned)(slot * (unsigned)p.D + c0) * sizeof(T);
    const char* z = (const char*)((const T*)p.z + at.b * p.zb);
    const char* q = (const char*)((const T*)p.q + at.b * p.qb);
    const char* dh = BWD ? (const char*)((const T*)p.dh + at.b * p.db) : nullptr;
    const char* hs = BWD ? (const char*)((const T*)p.h + at.b * p.T * p.D) : nullptr;
    char* out0 = p.out0 ? (char*)((T*)p.out0 + at.b * p.T * p.D) : nullptr;
    char* out1 = p.out1 ? (char*)((T*)p.out1 + at.b * p.T * p.D) : nullptr;
    const long k_end = min(p.T, (at.seg + 1) * p.seg_rows);
    const float* init = BWD ? p.dlast : p.h0;

    // R rows of every tensor; `t0`: the uniform row of row r of a tile (where the tile passes the end it need not exist: no lane reads it then)
    typedef SeqRaw<T, V> Raw;
    struct Rows { Raw z[R], q[R], d[BWD ? R : 1], h[BWD ? R : 1]; int f[R]; };
    auto row = [&](long k0, int r) __attribute__((always_inline)) { return BWD ? p.T - 1 - k0 - (TY * R - 1) + (R - 1 - r) : k0 + r; };
    // Whole tiles are read without a condition: the compiler then knows how many requests are younger than those it waits for, and the wait for a
    // tile is none for the one requested behind it, nor for the stores between.
    auto read = [&](Rows& w, long k0, bool whole) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long k = k0 + ty * R + r, t = BWD ? p.T - 1 - k : k, t0 = row(k0, r);
            if (!whole) {                                // no row: x -> x
                w.z[r] = w.q[r] = Raw{};
                if constexpr (BWD) w.d[r] = w.h[r] = Raw{};
                if (PACKED) w.f[r] = 0;
            }
            if (whole || k < k_end) {
                w.z[r] = seq_raw<T, V>((const T*)(z + t0 * p.zr * (long)sizeof(T) + oz));
                w.q[r] = seq_raw<T, V>((const T*)(q + t0 * p.qr * (long)sizeof(T) + oq));
                if constexpr (BWD) {
                    w.d[r] = seq_raw<T, V>((const T*)(dh + t0 * p.dr * (long)sizeof(T) + od));
                    w.h[r] = seq_raw<T, V>((const T*)(hs + (t0 - 1) * p.D * (long)sizeof(T) + (t > 0 ? oo : oo + (unsigned)p.D * (unsigned)sizeof(T))));
                }
                if (PACKED) w.f[r] = p.info[t];
            }
        }
    };
    const long k_begin = at.seg * p.seg_rows, wholes = (k_end - k_begin) / (TY * R);
    Rows now, next;
    if (wholes > 0) read(now, k_begin, true);

    float carry[V];
    zero(carry);                                         // (packed: a sequence's own state enters at its first row)
    if (!PACKED && init) seq_load<float, V>(init + at.b * p.D + c0, carry);
    int buf = 0;
    if (TY > 1 && at.seg > 0) {                          // the segments in front: slot ty composes a run of them, then the slots compose
        float A[V], H[V], in[V];
        int cut = 0;
        zero(A, 1.f);
        zero(H);
        const int per = (at.seg + TY - 1) / TY;
        {
#pragma unroll 2
            for (int s = ty * per; s < min(at.seg, (ty + 1) * per); ++s) {
                float a[V], h[V];
                const float* g = p.agg + ((at.b * p.segs + s) * 2) * p.D + c0;
                seq_load<float, V>(g, a);
                seq_load<float, V>(g + p.D, h);
                const bool c = PACKED && p.cuts[s];
                cut |= c;
#pragma unroll
                for (int v = 0; v < V; ++v) { H[v] = c ? h[v] : fmaf(a[v], H[v], h[v]); A[v] = c ? 0.f : A[v] * a[v]; }
            }
        }
        S::template wave_scan<PACKED>(A, H, cut, sums[0]);
        __syncthreads();
        S::template waves_apply<PACKED>(carry, in, sums[0], tx);
        buf = 1;
    }
    auto tile = [&](const long k0, bool whole) __attribute__((always_inline)) {
        float h[V];
        if constexpr (TY > 1) {
            float A[V], H[V], in[V];
            int cut = 0;
            zero(A, 1.f);
            zero(H);
#pragma unroll
            for (int r = 0; r < R; ++r) compose<BWD, PACKED, V>(A, H, cut, now.z[r], BWD ? now.d[BWD ? r : 0] : now.q[r], now.f[r], init, c0, p.D);
#pragma unroll
            for (int r = 0; r < R; ++r) { seq_hold(now.z[r]); if constexpr (BWD) seq_hold(now.d[r]); else seq_hold(now.q[r]); }
            S::template wave_scan<PACKED>(A, H, cut, sums[buf]);
            __syncthreads();                             // one barrier a tile: the next tile's sums go to the other buffer
            S::template waves_apply<PACKED>(carry, in, sums[buf], tx);
            buf ^= 1;
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = PACKED && cut ? H[v] : fmaf(A[v], in[v], H[v]);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = carry[v];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long k = k0 + ty * R + r, t = BWD ? p.T - 1 - k : k, out = row(k0, r) * p.D * (long)sizeof(T);
            if (!whole && k >= k_end) continue;
            const int f = PACKED ? now.f[r] : 0;
            const bool none = PACKED && f < 0, head = PACKED ? f >= 0 && (f & kFirst) : t == 0, tail = PACKED ? f >= 0 && (f & kLast) : t == p.T - 1;
            const long own = (PACKED ? (long)(f >> 2) : at.b) * p.D + c0;
            if (PACKED && (BWD ? tail : head)) { if (init) seq_load<float, V>(init + own, h); else zero(h); }
            if constexpr (!BWD) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = none ? 0.f : fmaf(1.f - now.z[r][v], h[v], now.z[r][v] * now.q[r][v]);
                seq_store<T, V>((T*)(out0 + out + oo), h, p.stream);
                if (tail && p.state) seq_store<float, V>(p.state + own, h);
            } else {
                float dz[V], dq[V], before[V];
#pragma unroll
                for (int v = 0; v < V; ++v) before[v] = now.h[r][v];
                if (head) { if (p.h0) seq_load<float, V>(p.h0 + own, before); else zero(before); }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float g = none ? 0.f : now.d[r][v] + h[v];
                    dz[v] = none ? 0.f : g * (now.q[r][v] - before[v]);
                    dq[v] = none ? 0.f : g * now.z[r][v];
                    h[v] = none ? 0.f : (1.f - now.z[r][v]) * g;
                }
                if (out0) seq_store<T, V>((T*)(out0 + out + oo), dz, p.stream);
                if (out1) seq_store<T, V>((T*)(out1 + out + oo), dq, p.stream);
                if (head && p.state) seq_store<float, V>(p.state + own, h);
            }
        }
        if constexpr (TY == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = h[v];
        }
    };
    for (long i = 0; i < wholes; ++i) {
        read(next, k_begin + min(i + 1, wholes - 1) * (TY * R), true);
        tile(k_begin + i * (TY * R), true);
        now = next;
    }
    if (k_begin + wholes * (TY * R) < k_end) {
        read(now, k_begin + wholes * (TY * R), false);
        tile(k_begin + wholes * (TY * R), false);
    }
}

// Packed rows: what each row is.  cu [S + 1] need not be sound for memory's sake: an owner is always one of the S sequences, and a sequence that
// would pass the last row ends there, one that would begin before the first row begins with it.  The workgroups behind those of the rows share the empty
// sequences: their states, which no row carries, are out = in (or 0).
__global__ __launch_bounds__(256) void gru_scan_rows_kernel(const int* __restrict__ cu, int S, int rows, int* __restrict__ info, int D, const float* __restrict__ in, float* __restrict__ out) {
    const long t = (long)blockIdx.x * 256 + threadIdx.x;
    const int row_groups = (rows + 255) / 256;
    if ((int)blockIdx.x >= row_groups) {
        for (int s = blockIdx.x - row_groups; s < S; s += gridDim.x - row_groups) {
            if (min(cu[s + 1], rows) > max(cu[s], 0)) continue;
            for (long c = threadIdx.x; c < D; c += 256) out[(long)s * D + c] = in ? in[(long)s * D + c] : 0.f;
        }
        return;
    }
    if (t >= rows) return;
    int lo = 0, hi = S + 1;                              // the first bound behind t
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (cu[m] <= t) lo = m + 1; else hi = m;
    }
    const int s = lo - 1;
    if (s < 0 || s >= S) { info[t] = -1; return; }
    info[t] = (s << 2) | (max(cu[s], 0) == t ? kFirst : 0) | (min(cu[s + 1], rows) == t + 1 ? kLast : 0);
}

struct Plan { int V, TX, TY, R, groups, segs; long seg_rows, workgroups; };
constexpr long kMostGroups = (1L << 24) - 1;             // a grid holds less than 2^32 threads
constexpr int kEmptyGroups = 1 << 20;                    // of the empty sequences, besides those of up to 2^31 rows

// Vectors of 16 bytes, single values for rows shorter than that.  TY = 1 (a lane walks the whole sequence, the lanes of all batches side by side) where the
// sequence is no longer than 16 rows or the channels alone would give every CU 16 workgroups of time slots; else 16 time slots, rows of 256 bytes (8 with single
// values, whose rows need more lanes to fill a cache line).  What counts are lanes that hold channels (training steps, us, slots or lanes): 512 x 8192 x 16 bf16, two
// lanes to a batch, 1495 or 8950; 512 x 4096 x 64 738 or 6190; 300 x 1000 x 1000 fp16 1530 or 2025; at the bound 512 x 24 x 1024 81 or 45, 512 x 100 x 1024 213 or 226,
// 512 x 2000 x 1000 fp32 11200 or 7730; 20000 x 100 x 8 fp32 337 or 205.  Rows of 64 lanes and more start at a multiple of 16, whole 256 bytes.
// Segments: forward as many as the chip holds workgroups of the second kernel at once, three to a CU (145 registers); backward 1024, which are held at once in fp32 (116 registers,
// four to a CU) and two rounds of two to a CU in 16 bits (170); none below two tiles (65536 x 1024 bf16, forward: 74 us with 768 workgroups, 85 us with 1024; backward:
// 212 with 768, 166 with 1024, 184 with 768 of two rows a slot).
int vec_of(int dtype, long D) { const int V = 16 / seq_size(dtype); return D < V ? 1 : V; }
Plan plan_of(int V, long B, long T, long D, bool bwd) {
    Plan p;
    p.V = V;
    const long lanes = (D + V - 1) / V;
    p.TY = V > 1 ? 16 : 8;
    p.TX = 256 / p.TY;
    p.R = 4;
    p.segs = 1;
    p.seg_rows = T;
    const long groups = (lanes + p.TX - 1) / p.TX;
    if (T <= 16 || B * groups * p.TX >= 256 * 256) {
        p.TY = 1;
        p.TX = 256;
        p.groups = (int)(lanes < 64 ? lanes : (lanes + 15) / 16 * 16);
        p.workgroups = (B * p.groups + 255) / 256;
        return p;
    }
    p.groups = (int)groups;
    const long tile = (long)p.TY * p.R, tiles = (T + tile - 1) / tile;
    long segs = (bwd ? 1024 : 768) / (B * groups);
    segs = segs < 1 ? 1 : segs > 128 ? 128 : segs;
    const long per = segs < 2 ? tiles : (tiles + segs - 1) / segs < 2 ? 2 : (tiles + segs - 1) / segs;
    p.segs = (int)((tiles + per - 1) / per);
    p.seg_rows = per * tile;
    p.workgroups = B * p.segs * groups;
    return p;
}

template <typename T, int V, bool BWD, bool PACKED>
void launch(const Plan& pl, const ScanArgs& a, hipStream_t s) {
    const unsigned grid = (unsigned)pl.workgroups;
    constexpr int TY = V > 1 ? 16 : 8, R = BWD ? 1 : PACKED ? 2 : 4;      // registers: backward holds four tensors, packed rows their meaning and a second start
    if (pl.TY == 1) { gru_scan_kernel<T, V, 256, 1, R, BWD, PACKED><<<grid, 256, 0, s>>>(a); return; }
    if (pl.segs > 1) gru_scan_segments_kernel<T, V, 256 / TY, TY, BWD, PACKED><<<grid, 256, 0, s>>>(a);
    gru_scan_kernel<T, V, 256 / TY, TY, R, BWD, PACKED><<<grid, 256, 0, s>>>(a);
}
template <typename T, bool BWD>
void launch_any(const Plan& pl, const ScanArgs& a, hipStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (a.info) { if (pl.V == 1) launch<T, 1, BWD, true>(pl, a, s); else launch<T, W, BWD, true>(pl, a, s); }
    else { if (pl.V == 1) launch<T, 1, BWD, false>(pl, a, s); else launch<T, W, BWD, false>(pl, a, s); }
}

// The workspace: the segments' (A, H), their cuts, the packed rows' meaning.
long agg_floats(const Plan& p, long B, long D) { return p.segs > 1 ? (B * p.segs * 2 * D + 3) & ~3L : 0; }
long cut_floats(const Plan& p, bool packed) { return packed && p.segs > 1 ? (p.segs + 3) & ~3 : 0; }

int run(bool bwd, int dtype, ScanArgs a, const int* cu, int S, float* ws, const float* empty_in, hipStream_t s) {
    const int V = vec_of(dtype, a.D);
    const Plan pl = plan_of(V, a.B, a.T, a.D, bwd);
    if (pl.workgroups > kMostGroups) return MOTIF_ELIMIT;
    if (pl.TY > 1) for (long stride : {a.zr, a.qr, a.dr, (long)a.D}) if (stride > 1L << 22) return MOTIF_ELIMIT;      // 128 rows x 4 bytes in 32 bits
    a.groups = pl.groups;
    a.segs = pl.segs;
    a.seg_rows = pl.seg_rows;
    a.stream = a.B * a.T * a.D * seq_size(dtype) >= kSeqStream;
    a.agg = ws;
    if (cu) {
        a.cuts = (int*)(ws + agg_floats(pl, a.B, a.D));
        int* info = (int*)(ws + agg_floats(pl, a.B, a.D) + cut_floats(pl, true));
        const unsigned grid = (unsigned)cdiv(a.T, 256) + (a.state ? S < kEmptyGroups ? S : kEmptyGroups : 0);
        if (grid) gru_scan_rows_kernel<<<grid, 256, 0, s>>>(cu, S, (int)a.T, info, a.D, empty_in, a.state);
        a.info = info;
    }
    if (a.T > 0)
        seq_dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (bwd) launch_any<T, true>(pl, a, s); else launch_any<T, false>(pl, a, s);
        });
    MOTIF_LAUNCH_CHECK();
    return MOTIF_OK;
}

int check_sizes(long B, long T, long D, int S, const void* cu, int dtype) {
    if (B < 1 || T < 0 || D < 1 || !seq_dtype_ok(dtype)) return MOTIF_EINVAL;
    if (cu ? (B != 1 || S < 1) : T < 1) return MOTIF_EINVAL;
    if (D > 0x0fffffffL || T > 0x7ffffff0L || B >= (1L << 29) || S >= (1 << 29)) return MOTIF_ELIMIT;
    return MOTIF_OK;
}
}  // namespace

extern "C" long motif_gru_scan_ws_floats(long B, long T, long D, int packed, int dtype) {
    const int rc = check_sizes(B, T, D, packed ? 1 : 0, packed ? (const void*)&B : nullptr, dtype);
    if (rc) return rc;
    long need = 0;                                       // of either direction
    for (bool bwd : {false, true}) {
        const Plan p = plan_of(vec_of(dtype, D), B, T, D, bwd);
        const long n = agg_floats(p, B, D) + cut_floats(p, packed);
        need = n > need ? n : need;
    }
    return need + (packed ? T : 0);
}

extern "C" int motif_gru_scan_fwd(const void* z, long z_bs, long z_rs, const void* q, long q_bs, long q_rs, const float* h0, const int32_t* cu_seqlens, int S,
                                  void* h, float* h_last, float* workspace, long B, long T, long D, int dtype, void* stream) {
    const int rc = check_sizes(B, T, D, S, cu_seqlens, dtype);
    if (rc) return rc;
    if ((T > 0 && (!z || !q || !h)) || z_bs < 0 || z_rs < 0 || q_bs < 0 || q_rs < 0) return MOTIF_EINVAL;
    if (!workspace && motif_gru_scan_ws_floats(B, T, D, cu_seqlens != nullptr, dtype) > 0) return MOTIF_EINVAL;
    ScanArgs a = {};
    a.z = z; a.q = q; a.h0 = h0; a.out0 = h; a.state = h_last;
    a.zb = z_bs; a.zr = z_rs; a.qb = q_bs; a.qr = q_rs;
    a.T = T; a.B = (int)B; a.D = (int)D;
    return run(false, dtype, a, cu_seqlens, S, workspace, h0, (hipStream_t)stream);
}

extern "C" int motif_gru_scan_bwd(const void* z, long z_bs, long z_rs, const void* q, long q_bs, long q_rs, const float* h0, const int32_t* cu_seqlens, int S,
                                  const void* h, const void* dh, long dh_bs, long dh_rs, const float* dh_last, void* dz, void* dq, float* dh0, float* workspace,
                                  long B, long T, long D, int dtype, void* stream) {
    const int rc = check_sizes(B, T, D, S, cu_seqlens, dtype);
    if (rc) return rc;
    if ((T > 0 && (!z || !q || !h || !dh)) || z_bs < 0 || z_rs < 0 || q_bs < 0 || q_rs < 0 || dh_bs < 0 || dh_rs < 0) return MOTIF_EINVAL;
    if (T > 0 && !dz && !dq && !dh0) return MOTIF_EINVAL;
    if (!workspace && motif_gru_scan_ws_floats(B, T, D, cu_seqlens != nullptr, dtype) > 0) return MOTIF_EINVAL;
    ScanArgs a = {};
    a.z = z; a.q = q; a.h = h; a.dh = dh; a.h0 = h0; a.dlast = dh_last; a.out0 = dz; a.out1 = dq; a.state = dh0;
    a.zb = z_bs; a.zr = z_rs; a.qb = q_bs; a.qr = q_rs; a.db = dh_bs; a.dr = dh_rs;
    a.T = T; a.B = (int)B; a.D = (int)D;
    return run(true, dtype, a, cu_seqlens, S, workspace, dh_last, (hipStream_t)stream);
}
