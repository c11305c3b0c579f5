// Gated feed-forward block: both projections, the activation and the product in one kernel, and its backward pass.
//
//   forward    G = x Wg^T + bg,  U = x Wu^T + bu,  h = act(G) * U
//   backward   dG = dh * U * act'(G),  dU = dh * act(G)
//              dx = dG Wg + dU Wu,   dWg = dG^T x,  dWu = dU^T x,   dbg, dbu = sums of dG, dU over the rows
//
// Three matrix products with two right-hand sides each, all bound by the matrix cores from a few hundred rows on.  One kernel serves them
// (gemm_kernel): C = sum over segments of A_s B_s with a tile's columns in two halves that come from two matrices -- the gate's and the up
// projection's (forward: the same columns of both, so that a wave holds G and U of the same outputs in its accumulators; weights'
// gradients: dG and dU) -- or are the two neighbouring runs of one (dx).  Either operand may lie with its reduction axis dense or across
// (transposed on the way from LDS to the registers), so every tensor is read as it lies.  fp32 runs on the same kernel: every operand is
// split exactly into three bf16 parts, and the six products that reach fp32's last place are six segments of the reduction.  Operands
// whose rows are not whole 16-byte pieces are laid out first (layout_kernel).
// G and U are kept in fp32 for the backward pass: rounded to the data's type they would add an error of their own to every gradient; dG and
// dU are rounded once, to be operands of the matrix cores: to 8 bits (bf16) or 11 (fp16), which makes the 16-bit gradients' rms error 1.4 times what fp32
// operands would leave (the outputs' own rounding is the rest); fp32 keeps all their bits.  fp16 ends at 65504 and loses bits below 2^-14, where the
// gradients need not: see scale_of.
// Up to 64 rows the forward pass is bound by reading the weights (rows_kernel, which small products share); layers of up to 64 inputs hold theirs in registers (narrow_*_kernel).
// Measured, 8192 x 2048 -> 2 x 5632 bf16: forward 313 us (1.21 PFLOP/s; the library's product of that size alone 352), 400 with G and U written
// besides (369 MB); dG and dU 147 (646 MB, 4.4 TB/s; past the caches: in them they would push out
// what the products read, 4 % of an fp32 backward pass), dx 278 (1.36 PFLOP/s; the library 291), dWg and dWu 296 + 16 (1.21 PFLOP/s; 356).
// Sums over rows and over the pieces of a split reduction are taken in a fixed order: no atomics, the same bits every time.
#include "seq_common.h"

namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSegs = 12;                                // dx in fp32: two pairs of operands, six products each

// ---- activations.  FAST: v_exp_f32 and v_rcp_f32 as they are (relative error 2^-24 (|g| + 4), behind a rounding to 8 or 11 bits); else
// expf and a reciprocal with a Newton step, one division's worth of accuracy at a third of its instructions ---------------------------------------
template <bool FAST>
__device__ __forceinline__ float reciprocal(float d) {  // finite d
    const float t = __builtin_amdgcn_rcpf(d);
    return FAST ? t : fmaf(t, fmaf(-d, t, 1.f), t);
}
// s = 1 / (1 + exp(-g)) and `rest` = 1 - s, both from e = exp(-|g|): neither passes a type's range, nor is one a difference from 1.
template <bool FAST>
__device__ __forceinline__ float sigm(float g, float& rest) {
    const float e = FAST ? __expf(-fabsf(g)) : expf(-fabsf(g)), t = reciprocal<FAST>(1.f + e), u = e * t;
    rest = g < 0.f ? t : u;
    return g < 0.f ? u : t;
}
// Phi(g) = erfc(-g / sqrt 2) / 2, and E = exp(-g^2 / 2).  erfc(x) exp(x^2) is smooth and falls like 1 / x: as t P(t) with t = 1 / (1 + 0.35 |g|), P of degree 8
// fitted to the least relative error, it is off by 6.2e-8 of itself and 2.9e-8 of 1 over |g| <= 14 (below, E is 0).  No difference of near values on the negative side, and
// E serves the derivative.  E is off by 2^-23.9 of 1 at most, of itself by (1.2 g^2 + 2) 2^-24 -- the square and its product with log2 e are rounded --: gelu(-5) by up to 40 x
// 2^-24 of itself (as (1 + erf) / 2 in fp32 it would be a difference with 2^-24 of 1 left, a tenth of its value).
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float g, float& E) {
    const float t = reciprocal<FAST>(fmaf(0.35f, fminf(fabsf(g), 64.f), 1.f));
    float p = -0.0291459057f;
    p = fmaf(p, t, 0.143971592f);
    p = fmaf(p, t, -0.255714029f);
    p = fmaf(p, t, 0.159173936f);
    p = fmaf(p, t, -0.0231096949f);
    p = fmaf(p, t, 0.105507948f);
    p = fmaf(p, t, 0.119832881f);
    p = fmaf(p, t, 0.139861867f);
    p = fmaf(p, t, 0.139621407f);
    E = __expf(-0.5f * g * g);
    const float q = E * (p * t);
    return g < 0.f ? q : 1.f - q;
}
// v = act(g) and d = act'(g) of N values.  One branch for all of them: the values' chains of instructions then overlap.
template <bool FAST, int N>
__device__ __forceinline__ void gates(const float (&g)[N], int act, float (&v)[N]) {
    if (act == MOTIF_GATE_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float E;
            v[e] = g[e] * normal_cdf<FAST>(g[e], E);
        }
    } else {
        const bool silu = act == MOTIF_GATE_SILU;        // g s, or s
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float rest;
            v[e] = (silu ? g[e] : 1.f) * sigm<FAST>(g[e], rest);
        }
    }
}
template <bool FAST, int N>
__device__ __forceinline__ void gate_grads(const float (&g)[N], int act, float (&v)[N], float (&d)[N]) {
    if (act == MOTIF_GATE_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float E;
            const float phi = normal_cdf<FAST>(g[e], E);
            v[e] = g[e] * phi;
            d[e] = fmaf(g[e] * 0.39894228f, E, phi);
        }
    } else {
        const bool silu = act == MOTIF_GATE_SILU;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float rest;
            const float s = sigm<FAST>(g[e], rest), m = silu ? g[e] : 1.f;
            v[e] = m * s;
            d[e] = s * fmaf(m, rest, silu ? 1.f : 0.f);
        }
    }
}

// ---- the matrix product ------------------------------------------------------------------------------------------------------------------
// GATED  h = act(A B0^T + bias0) * (A B1^T + bias1), G and U to keep         A [M][K], B0, B1 [N][K]
// ONE    C = sum of A_s B_s                                                  A [M][K], B [K][N]: the halves are neighbouring columns of it
// TWO    C0^T = A^T B0, C1^T = A^T B1                                        A [K][M], B0, B1 [K][N], C0, C1 [N][M]: a lane then holds four
//                                                                           consecutive rows of A, the matrix instruction takes its operands the other way round
enum GemmMode { GATED, ONE, TWO };
struct GemmArgs {
    const void* a[kSegs];
    const void* b0[kSegs];
    const void* b1[kSegs];
    long lda, ldb;                                       // in elements, multiples of 8
    int nseg, units;                                     // segments; units of 64 of the reduction in each
    int ka, kb;                                          // reduction length of either operand's tensors: what lies behind it counts as zeros
    int M, N, wa, wb;                                    // output rows / columns of either half; ONE, TWO: columns of B, of A that may be read (multiples of 8)
    int tiles_m, tiles_n, whole, pieces, units_per_piece;   // tiles 0 .. whole - 1 are one workgroup's; the others' reductions are cut into pieces
    void *c0, *c1;                                       // outputs of type dtype, dense
    float *g, *u;                                        // GATED: [M][ldg], may be null
    long ldg;
    const void *bias0, *bias1;
    f32x4* part;                                         // pieces' accumulators: [tile - whole][piece][accumulator][thread]
    const float* up;                                     // ONE, TWO: what the outputs are multiplied by; null: 1
    int act, dtype;
};

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, bf16_t*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, f16_t*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 64 lanes x 16 bytes from global memory to `lds` .. + 1024: base + off of each lane, or an address of its own.  Written as assembly so that the
// compiler does not make every LDS read wait for all of them (it takes any for the one that fills what is read); the waits are counted by
// hand in the kernel.
__device__ __forceinline__ void to_lds(unsigned lds, const void* base, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void to_lds(unsigned lds, const void* own) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(lds), "v"(own) : "memory", "m0");
}
__device__ u32x4 g_zeros;                                // what lies behind the end of a reduction

template <typename T, typename O, int N>
__device__ __forceinline__ void store_run(void* p, long at, const float (&v)[N], int n) {      // n of N values; whole runs as one store, at any address
    O* o = (O*)p + at;
    if (n == N) seq_store<O, N>(o, v);
    else
#pragma unroll
        for (int i = 0; i < N; ++i) if (i < n) o[i] = (O)v[i];
}
template <int N>
__device__ __forceinline__ void store_as(void* p, long at, const float (&v)[N], int n, int dtype) {
    if (dtype == MOTIF_F32) store_run<float, float, N>(p, at, v, n);
    else if (dtype == MOTIF_BF16) store_run<bf16_t, bf16_t, N>(p, at, v, n);
    else store_run<f16_t, f16_t, N>(p, at, v, n);
}

// One operand of a tile: two blocks of C rows (of the output), 64 of the reduction deep, 128 C bytes each.  A wave requests two pieces of 1 KB of
// either block per unit.
//   dense     [C][64]: a piece is 8 rows of 128 bytes -- whole cache lines: rows of 64 bytes (units of 32) make twice the requests to L2, which then
//             bound the kernel.  The eight 16-byte pieces of a row are exchanged by a pattern of the row's number, so that the 16 rows x 16
//             bytes of a fragment's read lie in different banks.
//   across    [64][C]: a piece is 2 C bytes of 4 (C = 128) or 8 steps.  A fragment's read takes 32 bytes (16 rows) of 16 steps and turns them
//             in 4 x 4 steps (ds_read_b64_tr_b16: lane i of 16 gets row i of four steps); 32-byte pieces are exchanged by a pattern of the step.
template <bool ACROSS, int C>
struct Operand {
    static constexpr int kWaves = C / 16, kPieces = C / 8;                        // 16-byte pieces of an across row
    static __device__ __forceinline__ int across_swap(int k) { return C == 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2); }
    // piece i of this lane: its first step of a unit, its byte offset from (row `at` of the matrix, step 0); rows up to `most` exist
    static __device__ __forceinline__ void lane_of(int wave, int lane, int i, int first, int at, int most, long ld, int& step, unsigned& off) {
        if (!ACROSS) {
            const int r = (i * kWaves + wave) * 8 + (lane >> 3);
            step = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
            off = (unsigned)(min(first + r, most - 1) - at) * (unsigned)ld * 2u + (unsigned)step * 2u;
        } else {
            const int c = lane % kPieces;
            step = (i * kWaves + wave) * (64 / kPieces) + lane / kPieces;
            off = (unsigned)step * (unsigned)ld * 2u + (unsigned)(min(first + (((c >> 1) ^ across_swap(step)) * 2 + (c & 1)) * 8, most - 8) - at) * 2u;
        }
    }
    // this lane's byte of a fragment of half `kk` of a unit, but for its row
    static __device__ __forceinline__ int frag_of(int lane, int kk) {
        if (!ACROSS) return (lane & 15) * 128 + ((kk * 4 + (lane >> 4)) ^ ((lane >> 1) & 7)) * 16;
        return (kk * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2)) * (2 * C) + (lane & 3) * 8;
    }
    static __device__ __forceinline__ s16x8 read(const char* block, int frag, int row, int lane) {
        if constexpr (!ACROSS) return *(const s16x8*)(block + frag + row * 128);
        else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* P;
            // the pattern is that of the step, whatever its bits 2 and 5 are: the same for the second four steps and for either half
            const int piece = ((row >> 4) ^ across_swap((lane >> 4) * 8 + ((lane & 15) >> 2))) * 32;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(block + frag + piece)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(block + frag + piece + 8 * C));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// Where a tile lies.  Workgroups are dealt to the eight XCDs in turn: each XCD takes a contiguous run of tiles, column by column within bands of 8 tile
// rows, so that the tiles in flight on one XCD share their rows of both operands in its L2.
template <int C, GemmMode MODE>
struct Tile {
    int m0, n0[2];
    __device__ __forceinline__ Tile(const GemmArgs& p, int id) {
        const int tiles = p.tiles_m * p.tiles_n, xcd = id & 7, q = tiles >> 3, r = tiles & 7;
        id = xcd * q + (xcd < r ? xcd : r) + (id >> 3);
        const int band = id / (8 * p.tiles_n), in = id - band * 8 * p.tiles_n, bh = min(8, p.tiles_m - band * 8), tn = in / bh;
        m0 = (band * 8 + in % bh) * 2 * C;
        n0[0] = tn * (MODE == ONE ? 2 * C : C);
        n0[1] = MODE == ONE ? n0[0] + C : n0[0];
    }
};

// One fragment pair (i, j) of a wave's outputs: o0, o1 of the two halves.
template <int C, GemmMode MODE>
struct Store {
    const GemmArgs& p;
    const Tile<C, MODE>& t;
    int m, c, lo, hi;                                    // this wave's first row of A and column of a half; of a fragment: the lane's place
    float bias[2][2][4], up;                             // GATED: [half][j]
    __device__ __forceinline__ Store(const GemmArgs& p_, const Tile<C, MODE>& t_, int wave, int lane) : p(p_), t(t_) {
        constexpr int WN = C / 32;
        m = t.m0 + wave / WN * C;
        c = wave % WN * 32;
        lo = lane & 15;
        hi = (lane >> 4) * 4;
        up = MODE != GATED && p.up ? *p.up : 1.f;
        if constexpr (MODE == GATED) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = min(t.n0[0] + c + j * 16 + hi + e, p.N - 1);
                    bias[0][j][e] = p.bias0 ? seq_param(p.bias0, n, p.dtype) : 0.f;
                    bias[1][j][e] = p.bias1 ? seq_param(p.bias1, n, p.dtype) : 0.f;
                }
        }
    }
    __device__ __forceinline__ void operator()(int i, int j, const f32x4& o0, const f32x4& o1) const {
        if constexpr (MODE == GATED) {
            const int row = m + i * 16 + lo, n = t.n0[0] + c + j * 16 + hi, cnt = min(4, p.N - n);
            if (row >= p.M || cnt <= 0) return;
            float g[4], u[4], v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) { g[e] = o0[e] + bias[0][j][e]; u[e] = o1[e] + bias[1][j][e]; }
            if (p.dtype == MOTIF_F32) gates<false>(g, p.act, v); else gates<true>(g, p.act, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= u[e];
            store_as<4>(p.c0, (long)row * p.N + n, v, cnt, p.dtype);
            if (p.g) {                                   // (their rows are padded to whole runs)
                seq_store<float, 4>(p.g + row * p.ldg + n, g);
                seq_store<float, 4>(p.u + row * p.ldg + n, u);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int a = m + i * 16, n = t.n0[h] + c + j * 16;
                const int row = MODE == ONE ? a + lo : n + lo, col = MODE == ONE ? n + hi : a + hi;
                const int rows = MODE == ONE ? p.M : p.N, cols = MODE == ONE ? p.N : p.M, cnt = min(4, cols - col);
                if (row >= rows || cnt <= 0) continue;
                const f32x4& o = h ? o1 : o0;
                const float v[4] = {o[0] * up, o[1] * up, o[2] * up, o[3] * up};
                store_as<4>(MODE == ONE || h == 0 ? p.c0 : p.c1, (long)row * cols + col, v, cnt, p.dtype);
            }
        }
    }
};

// Tile 2 C rows of A x C columns of either half of B; C / 16 waves (two along A), each C x 32 x 2 outputs.  The reduction advances in units of 64, two
// of which lie in LDS; the fragments of half a unit are read from LDS while those before them are multiplied.  One barrier a unit, in its middle:
// behind it every wave has the unit's second half in registers, so the unit after next may be requested into its place, and the next one is whole.
template <typename T, int C, GemmMode MODE>
__global__ __launch_bounds__(C * 4) void gemm_kernel(GemmArgs p) {
    constexpr int NW = C / 16, WN = NW / 2, MF = C / 16, HF = 2, BLOCK = C * 128, STAGE = 4 * BLOCK;
    using A = Operand<MODE == TWO, C>;
    using B = Operand<MODE != GATED, C>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    int id = blockIdx.x, part = -1;
    if (id >= p.whole && p.pieces > 1) { part = id - p.whole; id = p.whole + part / p.pieces; }
    const Tile<C, MODE> tile(p, id);
    const int m0 = tile.m0, n0[2] = {tile.n0[0], tile.n0[1]};
    const int am = MODE == TWO ? p.wa : p.M, bm = MODE != GATED ? p.wb : p.N;      // rows (columns) that may be read
    const int bat[2] = {n0[0], min(n0[1], bm - 8 < 0 ? 0 : bm - 8)};              // where the halves' pointers stand

    unsigned offa[2][2], offb[2][2];                     // [block][piece]
    int ka[2][2], kb[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            A::lane_of(wave, lane, i, m0 + h * C, m0, am, p.lda, ka[h][i], offa[h][i]);
            B::lane_of(wave, lane, i, n0[h], bat[h], bm, p.ldb, kb[h][i], offb[h][i]);
        }
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds + wave * 1024;
    const long unita = MODE == TWO ? 128 * p.lda : 128, unitb = MODE != GATED ? 128 * p.ldb : 128;      // bytes per unit
    const int enda = p.ka - (p.units - 1) * 64, endb = p.kb - (p.units - 1) * 64;  // what the last unit of a segment holds
    const bool ragged = enda < 64 || endb < 64;

    const int u_begin = part < 0 ? 0 : part % p.pieces * p.units_per_piece;
    const int count = part < 0 ? p.nseg * p.units : min(p.nseg * p.units - u_begin, p.units_per_piece);
    int seg = u_begin / p.units, left = p.units - (u_begin - seg * p.units);      // units left in the segment that is requested
    const char *pa, *pb0, *pb1;
    auto segment = [&](int unit) __attribute__((always_inline)) {
        pa = (const char*)p.a[seg] + (MODE == TWO ? m0 : (long)m0 * p.lda) * 2 + unit * unita;
        pb0 = (const char*)p.b0[seg] + (MODE != GATED ? bat[0] : (long)bat[0] * p.ldb) * 2 + unit * unitb;
        pb1 = (const char*)p.b1[seg] + (MODE != GATED ? bat[1] : (long)bat[1] * p.ldb) * 2 + unit * unitb;
    };
    segment(u_begin - seg * p.units);
    auto advance = [&]() __attribute__((always_inline)) {
        pa += unita; pb0 += unitb; pb1 += unitb;
        if (--left == 0 && seg + 1 < p.nseg) { ++seg; left = p.units; segment(0); }
    };
    auto piece = [&](int slot, int b, int i) __attribute__((always_inline)) {      // piece i of block b: A's two, B's two
        to_lds(lds0 + slot * STAGE + b * BLOCK + i * NW * 1024, b < 2 ? pa : b == 2 ? pb0 : pb1, b < 2 ? offa[b & 1][i] : offb[b & 1][i]);
    };
    auto request = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ragged && left == 1) {
                    const bool in = b < 2 ? ka[b & 1][i] < enda : kb[b & 1][i] < endb;
                    const char* own = b < 2 ? pa + offa[b & 1][i] : (b == 2 ? pb0 : pb1) + offb[b & 1][i];
                    to_lds(lds0 + slot * STAGE + b * BLOCK + i * NW * 1024, in ? own : (const char*)&g_zeros);
                } else piece(slot, b, i);
            }
        advance();
    };

    f32x4 acc[MF][2][HF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < HF; ++j) acc[i][h][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Frags { s16x8 a[MF], b[2][HF]; };
    const int fa[2] = {A::frag_of(lane, 0), A::frag_of(lane, 1)}, fb[2] = {B::frag_of(lane, 0), B::frag_of(lane, 1)};
    // a quarter of the fragments of half a unit / of its products
    auto fetch = [&](Frags& f, int slot, int kk, int q) __attribute__((always_inline)) {
        const char* st = lds + slot * STAGE;
        f.b[q >> 1][q & 1] = B::read(st + (2 + (q >> 1)) * BLOCK, fb[kk], wn * 32 + (q & 1) * 16, lane);
#pragma unroll
        for (int i = q * MF / 4; i < (q + 1) * MF / 4; ++i) f.a[i] = A::read(st + wm * BLOCK, fa[kk], i * 16, lane);
    };
    auto multiply = [&](const Frags& f, int q) __attribute__((always_inline)) {
#pragma unroll
        for (int i = q * MF / 4; i < (q + 1) * MF / 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < HF; ++j) acc[i][h][j] = MODE != TWO ? mfma(f.b[h][j], f.a[i], acc[i][h][j], (T*)nullptr) : mfma(f.a[i], f.b[h][j], acc[i][h][j], (T*)nullptr);
    };
    // Requests and reads are spread between the multiplications: issued in one go behind the barrier, by all waves at once, they hold up every wave's
    // first multiplication until the memory path and the LDS have taken all of them (measured: 500 of 1650 cycles per 32 of the reduction).
    auto spread = [&]() __attribute__((always_inline)) {
        constexpr int RA = MODE == TWO ? 2 : 1, RB = MODE != GATED ? 2 : 1, READS = RB + RA * MF / 4, MMAS = MF / 4 * 2 * HF, EACH = MMAS / READS;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                      // an LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);                   // matrix instructions
        }
        if constexpr (EACH * READS < MMAS) __builtin_amdgcn_sched_group_barrier(0x008, MMAS - EACH * READS, 0);
    };
    auto arrived = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    request(0);
    if (count > 1) {
        request(1);
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Frags f0, f1;                                        // of a unit's first and second half
#pragma unroll
    for (int q = 0; q < 4; ++q) fetch(f0, 0, 0, q);
    for (int u = 0; u < count; ++u) {
        for (int plain = min(count - 2 - u, left - (int)ragged); plain > 0; --plain, ++u) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                fetch(f1, u & 1, 1, q);
                multiply(f0, q);
                spread();
            }
            arrived();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                piece(u & 1, q, 0);
                piece(u & 1, q, 1);
                fetch(f0, (u + 1) & 1, 0, q);
                multiply(f1, q);
                spread();
            }
            advance();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) { fetch(f1, u & 1, 1, q); multiply(f0, q); }
        arrived();
        if (u + 2 < count) request(u & 1);
        if (u + 1 < count) {
#pragma unroll
            for (int q = 0; q < 4; ++q) fetch(f0, (u + 1) & 1, 0, q);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) multiply(f1, q);
    }

    if (part < 0) {
        const Store<C, MODE> store(p, tile, wave, lane);
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < HF; ++j) store(i, j, acc[i][0][j], acc[i][1][j]);
    } else {
        f32x4* o = p.part + ((long)part * (MF * 2 * HF)) * (C * 4) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < HF; ++j) o[((i * 2 + h) * HF + j) * (C * 4)] = acc[i][h][j];
    }
}

// The pieces of a tile's reduction, added in a fixed order, and the tile's outputs: a workgroup takes one fragment pair of all waves, its 1024 threads
// as groups of a tile's threads, each of which adds a run of the pieces.
template <int C, GemmMode MODE>
__global__ __launch_bounds__(1024) void join_kernel(GemmArgs p) {
    constexpr int MF = C / 16, TH = C * 4, GROUPS = 1024 / TH;
    __shared__ f32x4 sh[GROUPS - 1][2][TH];
    const int id = blockIdx.x / (MF * 2), i = blockIdx.x / 2 % MF, j = blockIdx.x % 2, tid = threadIdx.x % TH, group = threadIdx.x / TH;
    const int run = (p.pieces + GROUPS - 1) / GROUPS, k1 = min(p.pieces, (group + 1) * run);
    const f32x4* o = p.part + ((long)id * p.pieces * (MF * 4) + i * 4 + j) * TH + tid;
    f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
#pragma unroll 4
    for (int k = group * run; k < k1; ++k) {
        v0 += o[(long)k * (MF * 4) * TH];
        v1 += o[((long)k * (MF * 4) + 2) * TH];
    }
    if (group) { sh[group - 1][0][tid] = v0; sh[group - 1][1][tid] = v1; }
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 0; g < GROUPS - 1; ++g) { v0 += sh[g][0][tid]; v1 += sh[g][1][tid]; }
    const Tile<C, MODE> tile(p, p.whole + id);
    const Store<C, MODE> store(p, tile, __builtin_amdgcn_readfirstlane(tid >> 6), tid & 63);
    if (j == 0) store(i, 0, v0, v1); else store(i, 1, v0, v1);
}

// ---- laying operands out -----------------------------------------------------------------------------------------------------------------
// fp32 as three bf16 parts of 8 bits each, by truncation: x = p0 + p1 + p2 exactly (but for what is below bf16's smallest number).  An infinity or
// NaN has no further parts: their differences would make other NaNs of it.  An infinite operand multiplies every part of the other one, and times a
// part of 0 -- 1, 0.5, any value of few bits has such parts -- it would be a NaN where the product is infinite: a second or third part that comes out as
// 0 is bf16's smallest normal number of x's sign instead, 2^-36 of x at most (hence only from 2^-90 on: an infinity times less may come out as a NaN).
__device__ __forceinline__ void split3(float x, bf16_t (&out)[3]) {
    float r = x;
    const unsigned least = fabsf(x) >= 0x1p-90f ? (__builtin_bit_cast(unsigned, x) & 0x80000000u) | 0x00800000u : 0u;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const unsigned top = __builtin_bit_cast(unsigned, r) & 0xffff0000u;
        out[i] = __builtin_bit_cast(bf16_t, (unsigned short)((i && __builtin_bit_cast(float, top) == 0.f ? least : top) >> 16));
        r = (top & 0x7f800000u) == 0x7f800000u ? 0.f : r - __builtin_bit_cast(float, top);
    }
    // a NaN whose payload lies in the lower half only must not become an infinity
    if (x != x) out[0] = __builtin_bit_cast(bf16_t, (unsigned short)0x7fc0);
}
// eight values: one plane of T, or three of bf16, `plane` elements apart
__device__ __forceinline__ void put8(float* /*type*/, void* dst, long plane, long at, const float (&v)[8], bool stream = false) {
    float o[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bf16_t s[3];
        split3(v[e], s);
#pragma unroll
        for (int i = 0; i < 3; ++i) o[i][e] = (float)s[i];
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) seq_store<bf16_t, 8>((bf16_t*)dst + i * plane + at, o[i], stream);
}
__device__ __forceinline__ void put8(bf16_t*, void* dst, long, long at, const float (&v)[8], bool stream = false) { seq_store<bf16_t, 8>((bf16_t*)dst + at, v, stream); }
__device__ __forceinline__ void put8(f16_t*, void* dst, long, long at, const float (&v)[8], bool stream = false) { seq_store<f16_t, 8>((f16_t*)dst + at, v, stream); }

// src [rows][cols] with row stride rs -> dst rows of ld = cols rounded up to 8, zeros behind the last value of a row.  Eight values per thread.
template <typename T>
__global__ __launch_bounds__(256) void layout_kernel(const T* __restrict__ src, long rs, int rows, int cols, void* dst, long plane, int ld) {
    const int per = ld / 8;
    const long n = (long)rows * per;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / per;
        const int c = (int)(i - r * per) * 8;
        float v[8];
        if (c + 8 <= cols) seq_load<T, 8>(src + r * rs + c, v);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? (float)src[r * rs + c + e] : 0.f;
        put8((T*)nullptr, dst, plane, r * ld + c, v);
    }
}

// fp16: dG and dU are made and rounded as they are; where their largest finite value (`peak`) then passes fp16's range, or lies so low that what is 2^-10 of
// it no longer has all of its bits, they are made again times a power of two that takes the peak to 2^14 .. 2^15, and the products are multiplied by its
// reciprocal in fp32.  A gradient comes out infinite only where it is, and a small one keeps its bits.  Every workgroup writes its peak; the launch that
// makes them again reads all of them and ends at once if there is nothing to do: 4 to 9 us (training passes: 1337 x 1000 -> 2 x 2730 114 -> 120 us, 57600 x 64 -> 2 x 256 96 -> 101,
// 8192 x 2048 -> 2 x 5632 1165 -> 1173; made again: 136, 148).
template <typename T> constexpr bool kRanged = std::is_same_v<T, f16_t>;
__device__ __forceinline__ float peak_of(float peak, const float (&g)[8], const float (&u)[8]) {
    float most = 0.f;                                    // (fmaxf passes NaN by)
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(fmaxf(most, fabsf(g[e])), fabsf(u[e]));
    if (most < HUGE_VALF) return fmaxf(peak, most);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (fabsf(g[e]) < HUGE_VALF) peak = fmaxf(peak, fabsf(g[e]));
        if (fabsf(u[e]) < HUGE_VALF) peak = fmaxf(peak, fabsf(u[e]));
    }
    return peak;
}
template <int WAVES>
__device__ __forceinline__ float peak_in_workgroup(float peak, float* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = peak;
    __syncthreads();
    peak = sh[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) peak = fmaxf(peak, sh[i]);
    return peak;
}
// The power of two, from the n peaks that the first launch wrote; its reciprocal to peaks[n].
template <int WAVES>
__device__ __forceinline__ float scale_of(float* peaks, int n, float* sh) {
    float peak = 0.f;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += WAVES * 64) peak = fmaxf(peak, peaks[i]);
    peak = peak_in_workgroup<WAVES>(peak, sh);
    int e = 0;
    if (peak > 65504.f || (peak > 0.f && peak < 0x1p-4f)) e = max(-100, min(100, 14 + 127 - (int)(__builtin_bit_cast(unsigned, peak) >> 23)));
    if (blockIdx.x == 0 && threadIdx.x == 0) peaks[n] = __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
    return __builtin_bit_cast(float, (unsigned)(127 + e) << 23);
}

// dG and dU: [rows][ld], ld = F rounded up to 8 (G and U have it too), zeros behind F; fp32: three planes.  dU lies `pair` elements behind dG.
// A workgroup takes 256 columns x `rows` rows, eight columns per thread, and sums its columns over its rows (part [row blocks][2][F], may be null).
// `id`: the workgroup's place, one of `blocks`.  AGAIN: a workgroup takes several, times scale_of.
template <typename T, bool AGAIN>
__device__ __forceinline__ void gate_grad_block(const int id, const float scale, float& peak, float (&sh)[8][2][32][9], const T* __restrict__ dh, long dhs, const float* __restrict__ G,
                                                const float* __restrict__ U, int M, int F, int ld, int act, void* dst, long plane, long pair, float* part, int rows, bool stream) {
    using O = std::conditional_t<sizeof(T) == 4, bf16_t, T>;
    const int cols = (ld + 255) / 256, cb = id % cols, rb = id / cols;      // neighbouring workgroups take neighbouring columns of the same rows
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c0 = cb * 256 + x * 8, c = min(c0, ld - 8);
    const long r0 = (long)rb * rows;
    float sg[8], su[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
    // Every access is taken (rows behind the last do it again, lanes behind the last columns theirs, for no sum): the next row's requests then
    // stay in flight while this one is computed and written.
    struct Row { SeqRaw<T, 8> d; SeqRaw<float, 8> g, u; };
    auto read = [&](Row& w, long r) __attribute__((always_inline)) {
        const T* at = dh + r * dhs + c;
        if (F >= 8) w.d = seq_raw<T, 8>(at - max(c + 8 - F, 0));      // a run that passes the row's end: the row's last eight values, moved below
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) w.d.v[e] = c + e < F ? at[e] : (T)0.f;
        w.g = seq_raw<float, 8>(G + r * ld + c);
        w.u = seq_raw<float, 8>(U + r * ld + c);
    };
    const int move = F >= 8 ? max(c + 8 - F, 0) : 0;     // 0 but in the last run
    Row now, next;
    read(now, min(r0 + y, (long)M - 1));
    for (int i = y; i < rows; i += 8) {
        const long r = min(r0 + i, (long)M - 1);
        const bool counts = r0 + i < M && c == c0;
        read(next, min(r0 + min(i + 8, rows - 8 + y), (long)M - 1));
        float g[8], u[8], d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = now.d[e];
        if (move) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {                // d[e] = what stands at e + move (a run-time index would put the values into memory)
                float t = 0.f;
#pragma unroll
                for (int k = e; k < 8; ++k) t = k == e + move ? now.d[k] : t;
                d[e] = t;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = now.g[e];
        float v[8], dv[8];
        gate_grads<sizeof(T) == 2>(g, act, v, dv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g[e] = c + e < F ? d[e] * now.u[e] * dv[e] : 0.f;
            u[e] = c + e < F ? d[e] * v[e] : 0.f;
            sg[e] += counts ? g[e] : 0.f;
            su[e] += counts ? u[e] : 0.f;
            if constexpr (AGAIN) { g[e] *= scale; u[e] *= scale; }
        }
        if constexpr (kRanged<T> && !AGAIN) peak = peak_of(peak, g, u);
        put8((T*)nullptr, dst, plane, r * ld + c, g, stream);
        put8((T*)nullptr, (O*)dst + pair, plane, r * ld + c, u, stream);
        now = next;
    }
    if (AGAIN || !part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) { sh[y][0][x][e] = sg[e]; sh[y][1][x][e] = su[e]; }
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int k = i >> 8, cx = i & 255, cc = cb * 256 + cx;
        if (cc >= F) continue;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += sh[q][k][cx >> 3][cx & 7];
        part[((long)rb * 2 + k) * F + cc] = s;
    }
}
template <typename T, bool AGAIN>
__global__ __launch_bounds__(256) void gate_grad_kernel(const T* __restrict__ dh, long dhs, const float* __restrict__ G, const float* __restrict__ U, int M, int F, int ld, int act,
                                                       void* dst, long plane, long pair, float* part, int rows, bool stream, float* peaks, int blocks) {
    __shared__ float sh[8][2][32][9], waves[4];
    float peak = 0.f;
    if constexpr (!AGAIN) {
        gate_grad_block<T, false>(blockIdx.x, 1.f, peak, sh, dh, dhs, G, U, M, F, ld, act, dst, plane, pair, part, rows, stream);
        if constexpr (kRanged<T>) {
            peak = peak_in_workgroup<4>(peak, waves);
            if (threadIdx.x == 0) peaks[blockIdx.x] = peak;
        }
    } else {
        const float scale = scale_of<4>(peaks, blocks, waves);
        if (scale == 1.f) return;
        for (int id = blockIdx.x; id < blocks; id += gridDim.x) gate_grad_block<T, true>(id, scale, peak, sh, dh, dhs, G, U, M, F, ld, act, dst, plane, pair, part, rows, stream);
    }
}

// ---- few rows, small products -------------------------------------------------------------------------------------------------------------
// 16 MT rows to a workgroup, which takes 16 columns of both projections; its 8 waves share the reduction, each lane reads 32 bytes of a weight row at a time
// (16 rows x 128 bytes: whole cache lines) straight into the matrix instruction's operands -- which of the reduction's values a lane holds is free as
// long as both operands agree --; the waves' sums meet in LDS in a fixed order.  Bound by the weights' bytes.  fp32 runs on the fp32 matrix instruction.
// One row through 2048 -> 2 x 5632 bf16: 11.4 us, of which the 46 MB take 7.5 at the rate of a long read.
template <typename T, int MT, bool STEPS>
__global__ __launch_bounds__(512) void rows_kernel(const T* __restrict__ x, long xs, const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ bg, const T* __restrict__ bu,
                                                   T* __restrict__ h, float* __restrict__ G, float* __restrict__ U, long ldg, int M, int K, int F, int act) {
    constexpr int V = 16 / sizeof(T), STEP = 8 * V, NW = 8;
    __shared__ float sh[NW][2][16 * MT][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lo = lane & 15, kq = (lane >> 4) * 2 * V;
    const int f0 = blockIdx.x * 16, fr = min(f0 + lo, F - 1), m0 = blockIdx.y * 16 * MT;
    const T* pg = wg + (long)fr * K + kq;
    const T* pu = wu + (long)fr * K + kq;
    const T* px[MT];
    f32x4 ag[MT], au[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        px[i] = x + (long)min(m0 + i * 16 + lo, M - 1) * xs + kq;
        ag[i] = au[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    typedef SeqRaw<T, V> Raw;
    auto multiply = [&](const Raw& a, const Raw& b, const Raw& c, int i) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 2) {
            const s16x8 cv = __builtin_bit_cast(s16x8, c);
            ag[i] = mfma(__builtin_bit_cast(s16x8, a), cv, ag[i], (T*)nullptr);
            au[i] = mfma(__builtin_bit_cast(s16x8, b), cv, au[i], (T*)nullptr);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                ag[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], c[e], ag[i], 0, 0, 0);
                au[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[e], c[e], au[i], 0, 0, 0);
            }
        }
    };
    // Steps requested together -- MT = 1, all that a wave has up to K = 2048 (16 bits) -- by two workgroups to a CU, or a step ahead by one.
    const int whole = K / STEP;
    int s = wave;
    if constexpr (!STEPS) {
        constexpr int AHEAD = MT == 1 ? 4 : MT == 2 ? 2 : 1;
        for (; s + (AHEAD - 1) * NW < whole; s += NW * AHEAD) {
            Raw a[AHEAD][2], b[AHEAD][2], c[AHEAD][2][MT];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int k = (s + j * NW) * STEP + t * V;
                    a[j][t] = seq_raw<T, V>(pg + k);
                    b[j][t] = seq_raw<T, V>(pu + k);
#pragma unroll
                    for (int i = 0; i < MT; ++i) c[j][t][i] = seq_raw<T, V>(px[i] + k);
                }
            __builtin_amdgcn_sched_barrier(0);               // (all of them requested before the first is used)
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < MT; ++i) multiply(a[j][t], b[j][t], c[j][t][i], i);
        }
    } else if (s < whole) {
        struct Step { Raw a[2], b[2], c[2][MT]; };
        auto request = [&](Step& w, int step) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int k = step * STEP + t * V;
                w.a[t] = seq_raw<T, V>(pg + k);
                w.b[t] = seq_raw<T, V>(pu + k);
#pragma unroll
                for (int i = 0; i < MT; ++i) w.c[t][i] = seq_raw<T, V>(px[i] + k);
            }
        };
        Step now, next;
        request(now, s);
        for (; s < whole; s += NW) {
            request(next, min(s + NW, whole - 1));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < MT; ++i) multiply(now.a[t], now.b[t], now.c[t][i], i);
            now = next;
        }
    }
    auto read = [&](const T* at, int k) __attribute__((always_inline)) {         // zeros behind the row's end
        if (kq + k + V <= K) return seq_raw<T, V>(at + k);
        Raw v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = kq + k + e < K ? at[k + e] : (T)0.f;
        return v;
    };
    for (; s * STEP < K; s += NW)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k = s * STEP + t * V;
            const Raw a = read(pg, k), b = read(pu, k);
#pragma unroll
            for (int i = 0; i < MT; ++i) multiply(a, b, read(px[i], k), i);
        }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {                    // lane: row lo, columns 4 (lane / 16) + e
            sh[wave][0][i * 16 + lo][(lane >> 4) * 4 + e] = ag[i][e];
            sh[wave][1][i * 16 + lo][(lane >> 4) * 4 + e] = au[i][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * MT; i += 512) {
        const int row = i >> 4, m = m0 + row, f = f0 + (i & 15);
        if (m >= M || f >= F) continue;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) { g += sh[w][0][row][i & 15]; u += sh[w][1][row][i & 15]; }
        if (bg) g += (float)bg[f];
        if (bu) u += (float)bu[f];
        float v[1];
        gates<sizeof(T) == 2, 1>({g}, act, v);
        h[(long)m * F + f] = (T)(v[0] * u);
        if (G) { G[m * ldg + f] = g; U[m * ldg + f] = u; }
    }
}

// ---- narrow layers -----------------------------------------------------------------------------------------------------------------------
// K <= 64: a wave holds the weights of 32 columns of both projections in its registers and walks over blocks of 16 rows; neither a tile of the output nor
// fp32's three parts pass through memory.  Four values of the reduction to a lane: one matrix instruction of 16 bits, four of fp32 (each takes one
// value of every lane; which of the reduction's values those are is free as long as both operands agree).
// 57600 x 64 -> 2 x 256 fp32, gelu, training: forward 71 us (64 at least; 205 MB; the products of 64 x 512 fp32 alone 24 us, 103 us through the tiles and their three
// parts), backward 103 + 11 us for the workgroups' sums (229 MB; products 48 us; 250 us through the tiles).  Of a SIMD's cycles in them the products
// take 53 %, the activations and operands 25 %, waits the rest; making the next block's gradients between the products, starting a SIMD's two waves half a
// block apart and serving one of them first each left the time as it was, so that the instructions of both kinds seem to share what they need.
// The e-th of them; consecutive instructions should have accumulators of their own: one that adds to its predecessor's waits for it.
template <typename T> constexpr int kFours = sizeof(T) == 4 ? 4 : 1;
template <typename T>
__device__ __forceinline__ f32x4 mfma4(const SeqRaw<T, 4>& a, const SeqRaw<T, 4>& b, f32x4 c, int e) {
    if constexpr (sizeof(T) == 4)
        return __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    else if constexpr (std::is_same_v<T, bf16_t>)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ SeqRaw<T, 4> four(float a, float b, float c, float d) { return {{(T)a, (T)b, (T)c, (T)d}}; }

// Forward, K a multiple of 4 and at most 16 KQ, F one of 8.  The weights are the instruction's rows, in the order that gives a lane eight neighbouring
// columns of one row of the output; a run that would pass the last column is the last eight ones again, a row behind the last one the last, written
// alike.
template <typename T, int KQ, bool KEEP>
__global__ __launch_bounds__(256) void narrow_fwd_kernel(const T* __restrict__ x, long xs, const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ bg, const T* __restrict__ bu,
                                                         T* __restrict__ h, float* __restrict__ G, float* __restrict__ U, int M, int K, int F, int act, int walkers) {
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), runs = (F + 31) / 32, f0 = id % runs * 32, walker = id / runs;
    if (walker >= walkers) return;
    SeqRaw<T, 4> w[2][2][KQ];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            const int k = 16 * j + 4 * hi;
            const long at = (long)(min(f0 + 8 * (lo >> 2), F - 8) + 4 * t + (lo & 3)) * K + min(k, K - 4);
            w[0][t][j] = k < K ? seq_raw<T, 4>(wg + at) : four<T>(0.f, 0.f, 0.f, 0.f);
            w[1][t][j] = k < K ? seq_raw<T, 4>(wu + at) : four<T>(0.f, 0.f, 0.f, 0.f);
        }
    const int c = min(f0 + 8 * hi, F - 8);
    float b[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { b[0][e] = bg ? (float)bg[c + e] : 0.f; b[1][e] = bu ? (float)bu[c + e] : 0.f; }
    SeqRaw<T, 4> next[KQ];
    auto request = [&](int block) __attribute__((always_inline)) {
        const T* at = x + (long)min(block * 16 + lo, M - 1) * xs;
#pragma unroll
        for (int j = 0; j < KQ; ++j) next[j] = seq_raw<T, 4>(at + min(16 * j + 4 * hi, K - 4));
    };
    const int blocks = (M + 15) / 16;
    request(walker);
    for (int block = walker; block < blocks; block += walkers) {
        f32x4 a[2][2];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int t = 0; t < 2; ++t) a[p][t] = f32x4{b[p][4 * t], b[p][4 * t + 1], b[p][4 * t + 2], b[p][4 * t + 3]};
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
            SeqRaw<T, 4> v = next[j];
            if (16 * j + 4 * hi >= K) v = four<T>(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int e = 0; e < kFours<T>; ++e)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int t = 0; t < 2; ++t) a[p][t] = mfma4<T>(w[p][t][j], v, a[p][t], e);
        }
        request(min(block + walkers, blocks - 1));
        const long at = (long)min(block * 16 + lo, M - 1) * F + c;
        float g[8], u[8], o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g[e] = a[0][e >> 2][e & 3];
            u[e] = a[1][e >> 2][e & 3];
        }
        gates<sizeof(T) == 2>(g, act, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= u[e];
        seq_store<T, 8>(h + at, o);
        if (KEEP) { seq_store<float, 8>(G + at, g); seq_store<float, 8>(U + at, u); }
    }
}

// Backward in one pass over dh, G and U: F a multiple of 8 up to 256, which is what a workgroup's eight waves hold in columns (training steps of 57600 x 64 fp32: 2 x 256 159 us,
// through the tiles 2 x 264 433, 2 x 512 570, 2 x 1024 1062), K one of 4 up to 16 KT.  A workgroup's eight waves take NC runs of 32 columns of 8 / NC
// blocks of 16 rows.  A wave makes dG and dU of its rows and columns, with a row to a lane as dx needs them, and turns them over through LDS for the weights'
// gradients, whose sums stay in its registers over all of its rows; the runs' shares of dx meet in LDS, in a fixed order.
template <typename T, int KT, bool DX, bool DW>
__global__ __launch_bounds__(512) void narrow_bwd_kernel(const T* __restrict__ x, long xs, const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ dh, long dhs,
                                                         const float* __restrict__ G, const float* __restrict__ U, T* __restrict__ dx, float* __restrict__ dw_part,
                                                         float* __restrict__ db_part, int M, int K, int F, int act, int nc, float* peaks, bool again) {
    __shared__ float waves[8];
    float scale = 1.f, peak = 0.f;                       // fp16: see scale_of
    if constexpr (kRanged<T>) if (again) {
        scale = scale_of<8>(peaks, gridDim.x, waves);
        if (scale == 1.f) return;
    }
    const float up = 1.f / scale;
    __shared__ __attribute__((aligned(16))) float turn[8][2][32][20];              // [column][row]; 16-byte rows, writes of a wave on all banks
    __shared__ __attribute__((aligned(16))) float shares[DX ? 2 : 1][8][DX ? KT * 4 : 1][68];
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nr = 8 / nc, sub = wave / nc, f0 = wave % nc * 32, c = min(f0 + 8 * hi, F - 8);
    const bool mine = f0 + 8 * hi < F;
    SeqRaw<T, 4> w[DX ? 2 : 1][DX ? KT : 1][2];          // row k, four of the lane's eight columns
    if constexpr (DX) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const long at = (long)(c + 4 * t + e) * K + min(16 * kt + lo, K - 1);
                    w[0][kt][t].v[e] = mine ? wg[at] : (T)0.f;
                    w[1][kt][t].v[e] = mine ? wu[at] : (T)0.f;
                }
    }
    f32x4 dw[2][2][KT];
    float db[2][2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            db[p][t] = 0.f;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) dw[p][t][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    SeqRaw<T, 8> nd;
    SeqRaw<float, 8> ng, nu;
    auto request = [&](int r0) __attribute__((always_inline)) {
        const long r = min(r0 + lo, M - 1), at = r * F + c;
        nd = seq_raw<T, 8>(dh + r * dhs + c);
        ng = seq_raw<float, 8>(G + at);
        nu = seq_raw<float, 8>(U + at);
    };
    const int step = (int)gridDim.x * nr * 16;
    int buf = 0;
    request((blockIdx.x * nr + sub) * 16);
    for (int base = blockIdx.x * nr * 16; base < M; base += step) {
        const int r0 = base + sub * 16;
        SeqRaw<T, 4> xv[KT];                             // rows 4 hi .. + 3 of column lo
        if constexpr (DW)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const T* at = x + (long)min(r0 + 4 * hi + e, M - 1) * xs;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) xv[kt].v[e] = at[min(16 * kt + lo, K - 1)];
            }
        const unsigned keep = mine && r0 + lo < M ? ~0u : 0u;      // (as bits: a choice between values would become a branch around their making)
        float g[8], u[8], v[8], d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = ng[e];
        gate_grads<sizeof(T) == 2>(g, act, v, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g[e] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, nd[e] * nu[e] * d[e]) & keep);
            u[e] = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, nd[e] * v[e]) & keep);
            if constexpr (kRanged<T>) { g[e] *= scale; u[e] *= scale; }
            turn[wave][0][8 * hi + e][lo] = g[e];
            turn[wave][1][8 * hi + e][lo] = u[e];
        }
        if constexpr (kRanged<T>) peak = peak_of(peak, g, u);
        request(min(r0 + step, M - 1));
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();                 // (a wave's own part of `turn`; the LDS takes a wave's accesses in order)
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if constexpr (DX) {
            SeqRaw<T, 4> og[2], ou[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                og[t] = four<T>(g[4 * t], g[4 * t + 1], g[4 * t + 2], g[4 * t + 3]);
                ou[t] = four<T>(u[4 * t], u[4 * t + 1], u[4 * t + 2], u[4 * t + 3]);
            }
            f32x4 a[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) a[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2 * kFours<T>; ++e)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) a[kt] = mfma4<T>(w[e & 1][kt][t], e & 1 ? ou[t] : og[t], a[kt], e >> 1);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) *(f32x4*)&shares[buf][wave][kt * 4 + hi][lo * 4] = a[kt];
        }
        if constexpr (DW)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) xv[kt].v[e] = r0 + 4 * hi + e < M ? xv[kt].v[e] : (T)0.f;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x4 v = *(const f32x4*)&turn[wave][p][16 * t + lo][4 * hi];
                db[p][t] += (v[0] + v[1]) + (v[2] + v[3]);
                const SeqRaw<T, 4> o = four<T>(v[0], v[1], v[2], v[3]);
                if constexpr (DW)
#pragma unroll
                    for (int e = 0; e < kFours<T>; ++e)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) dw[p][t][kt] = mfma4<T>(o, xv[kt], dw[p][t][kt], e);
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if constexpr (DX) {
            __syncthreads();                             // the other buffer's sums were taken before this
            const int pairs = nr * 16 * KT * 8;
            for (int i = 0; i < pairs; i += 512) {       // two values each; rows and columns behind the last: those again
                const int q = min(i + (int)threadIdx.x, pairs - 1), m = min(q / (KT * 8), M - 1 - base), k = min(q % (KT * 8) * 2, K - 2);
                float s[2] = {0.f, 0.f};
                for (int n = 0; n < nc; ++n) {
                    const float* at = &shares[buf][(m >> 4) * nc + n][k >> 2][(m & 15) * 4 + (k & 3)];
                    s[0] += at[0];
                    s[1] += at[1];
                }
                if constexpr (kRanged<T>) { s[0] *= up; s[1] *= up; }
                seq_store<T, 2>(dx + (long)(base + m) * K + k, s);
            }
            buf ^= 1;
        }
    }
    const long slot = (long)blockIdx.x * nr + sub;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float s = db[p][t] * up;
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            const int f = f0 + 16 * t;
            if (db_part && hi == 0 && f + lo < F) db_part[(slot * 2 + p) * F + f + lo] = s;
            if constexpr (DW)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
                        if (f + 4 * hi + e < F && 16 * kt + lo < K) dw_part[((slot * 2 + p) * F + f + 4 * hi + e) * K + 16 * kt + lo] = dw[p][t][kt][e] * up;
        }
    if constexpr (kRanged<T>) if (!again) {
        peak = peak_in_workgroup<8>(peak, waves);
        if (threadIdx.x == 0) peaks[blockIdx.x] = peak;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = 64;
// Products for rows_kernel: up to 64 rows (fp32: 128), and beyond them what its workgroups of 64 rows x 16 columns have done in two rounds of the chip -- four where the
// tiles' operands would have to be laid out first -- and 2^19 steps of a workgroup; the tiles of so small a product leave most CUs idle.  bf16, this
// kernel or tiles: 256 x 1024 -> 2 x 1024 (256 workgroups) 9 or 18 us, 512 x 256 -> 2 x 1024 (512) 8 or 9, 512 x 1024 -> 2 x 1024 (512, 2^19 steps) 13
// or 13, 1024 x 512 -> 2 x 1024 (1024) 15 or 11; fp32: 512 x 256 -> 2 x 1024 12 or 29, 2048 x 128 -> 2 x 512 (1024) 12 or 23, 257 x 1000 -> 2 x 2729
// (855, 1.6 x 2^19) 65 or 61, 8192 x 72 -> 2 x 512 (4096) 51 or 30.  fp32 up to 128 rows whatever the size, whose weights would be laid out for little: 128 x
// 4096 -> 2 x 8192 198 or 293, 128 x 2048 -> 2 x 5632 82 or 98; 192 x 2048 -> 2 x 5632 134 or 126.
bool few(long M, long K, long F, int dtype, bool laid_out) {
    const long groups = (long)cdiv(F, 16) * cdiv(M, 64);
    return M <= (dtype == MOTIF_F32 ? 2 * kFewRows : kFewRows) || (groups <= (laid_out ? 1024 : 512) && groups * K <= 1L << 19);
}
// Waves of narrow_fwd_kernel to a CU: more hide more of the reads, until their writes get in each other's way (57600 x 64 -> 2 x 1024 bf16: 88 us with 8, 83 with 12;
// with kept projections 200 and 206).
int narrow_waves(bool keep) { return keep ? 8 : 12; }
constexpr long kMostRows = 1L << 22;                    // offsets within a tile are 32 bits: 256 rows x this x 2 bytes
int up8(long n) { return (int)((n + 7) & ~7L); }
int units_of(long n) { return (int)((n + 63) / 64); }
long up16b(long bytes) { return (bytes + 255) & ~255L; }
int planes(int dtype) { return dtype == MOTIF_F32 ? 3 : 1; }

// A workspace that is measured (base null) or handed out.
struct Arena {
    char* base;
    long used;
    void* take(long bytes) { char* p = base ? base + used : nullptr; used += up16b(bytes); return p; }
};
// An operand: `n` planes, `plane` elements apart, rows of ld.
struct Image { const void* p; long plane; int ld, n; };
const void* plane_of(const Image& m, int i) { return (const char*)m.p + (long)i * m.plane * 2; }

template <typename T>
void layout(const void* src, long rs, long rows, int cols, const Image& to, hipStream_t s) {
    const long blocks = (rows * (to.ld / 8) + 255) / 256;
    layout_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>((const T*)src, rs, (int)rows, cols, (void*)to.p, to.plane, to.ld);
}

// The products of two operands' parts that reach fp32's last place, smallest first: 2^-16 each of (0,2) (1,1) (2,0), 2^-8 of (0,1) (1,0), (0,0).  The three left out
// take 0.7 x 2^-24 off a product on average (truncated parts have its sign), 1 x 2^-24 rms, 2^-21 at most (both mantissas just below 1 + 2^-7).
void segments(GemmArgs& g, const Image& a, const Image& b0, const Image& b1) {
    if (a.n == 1) {
        g.a[g.nseg] = a.p; g.b0[g.nseg] = b0.p; g.b1[g.nseg] = b1.p;
        ++g.nseg;
        return;
    }
    static const int pairs[6][2] = {{0, 2}, {1, 1}, {2, 0}, {0, 1}, {1, 0}, {0, 0}};
    for (auto& q : pairs) {
        g.a[g.nseg] = plane_of(a, q[0]); g.b0[g.nseg] = plane_of(b0, q[1]); g.b1[g.nseg] = plane_of(b1, q[1]);
        ++g.nseg;
    }
}

// The tiles behind the last whole round of the chip are cut along the reduction so that their pieces fill it: the accumulators of a round are 64 MB,
// written and read again in about as long as 24 units of a tile take (8192 x 2048 x 5632 bf16, weights' gradients: 352 tiles, 380 us in two rounds,
// 326 us with the second one cut in two).
struct GemmPlan { bool big; int tiles_m, tiles_n, whole, pieces, units_per_piece; };
GemmPlan plan_with(bool big, long M, long N, int halves, long units) {
    GemmPlan p;
    p.big = big;
    const int t = big ? 256 : 128;
    p.tiles_m = cdiv(M, t);
    p.tiles_n = cdiv(N, halves == 2 ? t / 2 : t);
    const long tiles = (long)p.tiles_m * p.tiles_n, slots = big ? 256 : 512, rest = tiles % slots;
    long pieces = rest ? slots / rest : 1;
    if (pieces > units / 8) pieces = units / 8;
    if (pieces < 2 || units * (pieces - 1) < 24 * pieces) pieces = 1;
    p.units_per_piece = (int)((units + pieces - 1) / pieces);
    p.pieces = (int)((units + p.units_per_piece - 1) / p.units_per_piece);
    p.whole = (int)(p.pieces > 1 ? tiles - rest : tiles);
    return p;
}
// Rounds of the chip that a plan takes, one of 512 tiles of 128 being half of one of 256 tiles of 256, and dearer for the same work: 8 %
// in whole rounds, counted as 20 % (8192 x 2048 x 5632: 6 rounds of 256 take 374 us, 11 of 128 436 us).
double rounds_of(const GemmPlan& p, long units) {
    const long tiles = (long)p.tiles_m * p.tiles_n, slots = p.big ? 256 : 512;
    const double r = p.pieces > 1 ? p.whole / slots + (double)p.units_per_piece / units + 24. / units : (double)cdiv(tiles, slots);
    return p.big ? r : 0.6 * r;
}
// Tiles of 256 x 256 (C = 128) where they give every CU at least one and no fewer of 128 x 128, of which a CU holds two, end sooner (2048 x 2048 x
// 5632 bf16: two rounds of 256, 97 us, or three of 128, 88 us; 8192 x 1024 x 4096: 131 or 140 us).  `keep`: under a reduction of up to 6 units the
// epilogue, which then writes the projections too, is most of the time, and two tiles on a CU, the one in its products while the other writes, hide
// it (57600 x 64 x 256 fp32: 91 us with tiles of 256, 82 us with 128; 16384 x 128 x 2048 bf16: 94 or 83 us; 8192 x 512 x 4096: 153 or 152 us).
GemmPlan gemm_plan(long M, long N, int halves, long units, bool keep) {
    const GemmPlan big = plan_with(true, M, N, halves, units), small = plan_with(false, M, N, halves, units);
    const bool few = (long)big.tiles_m * big.tiles_n < 256;
    return few || (keep && units <= 6) || rounds_of(small, units) < rounds_of(big, units) ? small : big;
}
long part_bytes(const GemmPlan& p) {
    const long cut = (long)p.tiles_m * p.tiles_n - p.whole;
    return cut * p.pieces * (p.big ? 4L * 256 * 256 : 4L * 128 * 128);
}

template <typename T, int C, GemmMode MODE>
void gemm_tiles(const GemmPlan& pl, const GemmArgs& g, hipStream_t s) {
    const int cut = pl.tiles_m * pl.tiles_n - pl.whole;
    gemm_kernel<T, C, MODE><<<(unsigned)(pl.whole + (long)cut * pl.pieces), C * 4, 0, s>>>(g);
    if (cut) join_kernel<C, MODE><<<cut * (C / 16) * 2, 1024, 0, s>>>(g);
}
template <typename T, GemmMode MODE>
void gemm(const GemmPlan& pl, GemmArgs& g, hipStream_t s) {
    g.tiles_m = pl.tiles_m; g.tiles_n = pl.tiles_n; g.whole = pl.whole; g.pieces = pl.pieces; g.units_per_piece = pl.units_per_piece;
    if (pl.big) gemm_tiles<T, 128, MODE>(pl, g, s);
    else gemm_tiles<T, 64, MODE>(pl, g, s);
}
template <GemmMode MODE>
void gemm_dtype(int dtype, const GemmPlan& pl, GemmArgs& g, hipStream_t s) {
    if (dtype == MOTIF_F16) gemm<f16_t, MODE>(pl, g, s);
    else gemm<bf16_t, MODE>(pl, g, s);
}

// Whether an operand can be read as it lies: 16-bit values, rows of whole 16-byte pieces at 16-byte addresses.
bool direct(const void* p, long rs, long cols, int dtype) { return dtype != MOTIF_F32 && cols % 8 == 0 && rs % 8 == 0 && rs <= kMostRows && seq_aligned(p, 16); }

int check_mlp(long M, long K, long F, int act, int dtype) {
    if (M < 0 || K < 1 || F < 1 || !seq_dtype_ok(dtype) || act < MOTIF_GATE_SIGMOID || act > MOTIF_GATE_GELU) return MOTIF_EINVAL;
    if (K > 65536 || F > 65536 || M > kMostRows) return MOTIF_ELIMIT;
    return MOTIF_OK;
}

template <typename T, int MT>
void few_rows(const void* x, long xs, const void* wg, const void* wu, const void* bg, const void* bu, void* h, float* G, float* U, int M, int K, int F, int act, hipStream_t s) {
    // fp32 from 17 rows on multiplies a long row's steps for long enough to cover the next one's requests alone (64 rows, 4096 -> 2 x 8192: 102 us, 133 with
    // steps together; 1024 -> 2 x 1024 18 and 19; 512 -> 2 x 2048 13 and 11; bf16 4096 -> 2 x 8192 55 and 47).
    auto* kernel = rows_kernel<T, MT, false>;
    if constexpr (sizeof(T) == 4 && MT > 1) if (K >= 1024) kernel = rows_kernel<T, MT, true>;
    kernel<<<dim3(cdiv(F, 16), cdiv(M, 16 * MT)), 512, 0, s>>>((const T*)x, xs, (const T*)wg, (const T*)wu, (const T*)bg, (const T*)bu, (T*)h, G, U, up8(F), M, K, F, act);
}

bool narrow(long K, long F) { return K <= 64 && K % 4 == 0 && F % 8 == 0; }
bool narrow_bwd(long K, long F) { return narrow(K, F) && F <= 256; }
int column_runs(long F) { return F > 128 ? 8 : F > 64 ? 4 : F > 32 ? 2 : 1; }       // of 32 columns, of a workgroup's eight waves
int narrow_groups(long M, long F) {                      // one per CU; two blocks of rows each, so that the second is read while the first is computed
    const long n = cdiv(M, 2 * 16 * (8 / column_runs(F)));
    return (int)(n < 256 ? n : 256);
}
template <typename T>
void narrow_fwd(const void* x, long xs, const void* wg, const void* wu, const void* bg, const void* bu, void* h, float* G, float* U, int M, int K, int F, int act, hipStream_t s) {
    const int runs = (F + 31) / 32, blocks = (M + 15) / 16;
    int walkers = 256 * narrow_waves(G != nullptr) / runs;
    walkers = walkers < 1 ? 1 : walkers > blocks ? blocks : walkers;
    const unsigned grid = (unsigned)(((long)runs * walkers + 3) / 4);
    auto* kernel = K <= 32 ? G ? narrow_fwd_kernel<T, 2, true> : narrow_fwd_kernel<T, 2, false> : G ? narrow_fwd_kernel<T, 4, true> : narrow_fwd_kernel<T, 4, false>;
    kernel<<<grid, 256, 0, s>>>((const T*)x, xs, (const T*)wg, (const T*)wu, (const T*)bg, (const T*)bu, (T*)h, G, U, M, K, F, act, walkers);
}
template <typename T, int KT>
void narrow_bwd(int grid, const void* x, long xs, const void* wg, const void* wu, const void* dh, long dhs, const float* G, const float* U, void* dx, float* dw_part, float* db_part,
                float* peaks, int M, int K, int F, int act, hipStream_t s) {
    auto* kernel = dx && dw_part ? narrow_bwd_kernel<T, KT, true, true> : dx ? narrow_bwd_kernel<T, KT, true, false>
                 : dw_part ? narrow_bwd_kernel<T, KT, false, true> : narrow_bwd_kernel<T, KT, false, false>;
    for (bool again : {false, true})
        if (!again || (kRanged<T> && (dx || dw_part)))
            kernel<<<grid, 512, 0, s>>>((const T*)x, xs, (const T*)wg, (const T*)wu, (const T*)dh, dhs, G, U, (T*)dx, dw_part, db_part, M, K, F, act, column_runs(F), peaks, again);
}

// x, Wg and Wu as the products read them: as they lie, or laid out in the workspace.
struct Inputs { Image x, wg, wu; bool lay_x, lay_w; };
Inputs inputs_of(Arena& ws, const void* x, long xs, const void* wg, const void* wu, long M, long K, long F, int dtype) {
    Inputs f;
    const int n = planes(dtype), ld = up8(K);
    f.lay_x = !direct(x, xs, K, dtype);
    f.lay_w = !direct(wg, K, K, dtype) || !direct(wu, K, K, dtype);
    f.x = f.lay_x ? Image{ws.take(2 * n * M * ld), M * ld, ld, n} : Image{x, 0, (int)xs, 1};
    f.wg = f.lay_w ? Image{ws.take(2 * n * F * ld), F * ld, ld, n} : Image{wg, 0, (int)K, 1};
    f.wu = f.lay_w ? Image{ws.take(2 * n * F * ld), F * ld, ld, n} : Image{wu, 0, (int)K, 1};
    return f;
}
void lay_out(const Inputs& f, bool need_x, bool need_w, const void* x, long xs, const void* wg, const void* wu, long M, long K, long F, int dtype, hipStream_t s) {
    seq_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (f.lay_x && need_x) layout<T>(x, xs, M, (int)K, f.x, s);
        if (f.lay_w && need_w) { layout<T>(wg, K, F, (int)K, f.wg, s); layout<T>(wu, K, F, (int)K, f.wu, s); }
    });
}

// Rows of a workgroup of gate_grad_kernel: 16 -- the last round of many short workgroups leaves little of the chip idle (8192 x 5632 bf16 from memory: 147 us,
// 161 with 64 rows, whose column sums cost 5 us less; whole backward passes 0 to 2 % shorter) --, 8 where that would leave less than four per CU.
int grad_rows(long M, long F) { return (long)cdiv(M, 16) * cdiv(F, 256) < 1024 ? 8 : 16; }
long products(int dtype) { return planes(dtype) == 3 ? 6 : 1; }
GemmPlan fwd_plan(long M, long K, long F, int dtype, bool keep) { return gemm_plan(M, F, 2, products(dtype) * units_of(K), keep); }
GemmPlan dx_plan(long M, long K, long F, int dtype) { return gemm_plan(M, K, 1, 2 * products(dtype) * units_of(F), false); }
GemmPlan dw_plan(long M, long K, long F, int dtype) { return gemm_plan(K, F, 2, products(dtype) * units_of(M), false); }

int grad_blocks(long M, long F) { return (int)((long)cdiv(M, grad_rows(M, F)) * cdiv(up8(F), 256)); }
struct Backward { Inputs in; Image dg, du; float *bias_part, *peaks; f32x4* part; GemmPlan dx, dw; float* dw_part; bool one_pass; };
Backward backward_of(Arena& ws, const void* x, long xs, const void* wg, const void* wu, long M, long K, long F, int dtype, bool need_x, bool need_w, bool need_b) {
    Backward b = {};
    const int n = planes(dtype), ld = up8(F);
    if (narrow_bwd(K, F)) {
        b.one_pass = true;
        const long slots = (long)narrow_groups(M, F) * (8 / column_runs(F));
        if (need_w) b.dw_part = (float*)ws.take(4 * slots * 2 * F * K);
        if (need_b) b.bias_part = (float*)ws.take(4 * slots * 2 * F);
        if (dtype == MOTIF_F16) b.peaks = (float*)ws.take(4 * (narrow_groups(M, F) + 1));
        return b;
    }
    b.in = inputs_of(ws, x, xs, wg, wu, M, K, F, dtype);
    char* p = (char*)ws.take(2L * 2 * n * M * ld);
    b.dg = {p, M * ld, ld, n};
    b.du = {p ? p + 2L * n * M * ld : nullptr, M * ld, ld, n};
    if (need_x) b.dx = dx_plan(M, K, F, dtype);
    if (need_w) b.dw = dw_plan(M, K, F, dtype);
    if (need_b) b.bias_part = (float*)ws.take(4L * cdiv(M, grad_rows(M, F)) * 2 * F);
    if (dtype == MOTIF_F16) b.peaks = (float*)ws.take(4L * (grad_blocks(M, F) + 1));
    long part = need_x ? part_bytes(b.dx) : 0;           // the two products run one behind the other: one piece of memory serves both
    if (need_w && part_bytes(b.dw) > part) part = part_bytes(b.dw);
    if (part) b.part = (f32x4*)ws.take(part);
    return b;
}
}  // namespace

extern "C" long motif_gated_mlp_ws_bytes(const void* x, long x_rs, const void* w_gate, const void* w_up, long M, long K, long F, int dtype) {
    const int rc = check_mlp(M, K, F, MOTIF_GATE_SILU, dtype);
    if (rc) return rc;
    if (M <= kFewRows || narrow(K, F)) return 0;
    Arena ws = {nullptr, 0};
    const Inputs f = inputs_of(ws, x, x_rs, w_gate, w_up, M, K, F, dtype);
    if (few(M, K, F, dtype, f.lay_x || f.lay_w)) return 0;
    const long p0 = part_bytes(fwd_plan(M, K, F, dtype, false)), p1 = part_bytes(fwd_plan(M, K, F, dtype, true));
    ws.take(p0 > p1 ? p0 : p1);
    return ws.used;
}

extern "C" int motif_gated_mlp_fwd(const void* x, long x_rs, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, void* h, float* G, float* U,
                                   void* workspace, long M, long K, long F, int act, int dtype, void* stream) {
    const int rc = check_mlp(M, K, F, act, dtype);
    if (rc) return rc;
    if (M == 0) return MOTIF_OK;
    if (!x || !w_gate || !w_up || !h || x_rs < 0 || !G != !U) return MOTIF_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    if (M > kFewRows && narrow(K, F)) {
        seq_dispatch(dtype, [&](auto* t) { narrow_fwd<std::remove_pointer_t<decltype(t)>>(x, x_rs, w_gate, w_up, b_gate, b_up, h, G, U, (int)M, (int)K, (int)F, act, s); });
        MOTIF_LAUNCH_CHECK();
        return MOTIF_OK;
    }
    Arena ws = {(char*)workspace, 0};
    const Inputs f = inputs_of(ws, x, x_rs, w_gate, w_up, M, K, F, dtype);
    if (few(M, K, F, dtype, f.lay_x || f.lay_w)) {
        seq_dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (M <= 16) few_rows<T, 1>(x, x_rs, w_gate, w_up, b_gate, b_up, h, G, U, (int)M, (int)K, (int)F, act, s);
            else if (M <= 32) few_rows<T, 2>(x, x_rs, w_gate, w_up, b_gate, b_up, h, G, U, (int)M, (int)K, (int)F, act, s);
            else few_rows<T, 4>(x, x_rs, w_gate, w_up, b_gate, b_up, h, G, U, (int)M, (int)K, (int)F, act, s);
        });
        MOTIF_LAUNCH_CHECK();
        return MOTIF_OK;
    }
    const GemmPlan plan = fwd_plan(M, K, F, dtype, G != nullptr);
    f32x4* part = (f32x4*)ws.take(part_bytes(plan));
    if (ws.used && !workspace) return MOTIF_EINVAL;
    lay_out(f, true, true, x, x_rs, w_gate, w_up, M, K, F, dtype, s);
    GemmArgs g = {};
    segments(g, f.x, f.wg, f.wu);
    g.lda = f.x.ld; g.ldb = f.wg.ld;
    g.ka = g.kb = up8(K);
    g.units = units_of(K);
    g.M = (int)M; g.N = (int)F;
    g.c0 = h; g.g = G; g.u = U; g.ldg = up8(F); g.bias0 = b_gate; g.bias1 = b_up;
    g.act = act; g.dtype = dtype;
    g.part = part;
    gemm_dtype<GATED>(dtype, plan, g, s);
    MOTIF_LAUNCH_CHECK();
    return MOTIF_OK;
}

extern "C" long motif_gated_mlp_bwd_ws_bytes(const void* x, long x_rs, const void* w_gate, const void* w_up, long M, long K, long F, int dtype, int need_x, int need_w, int need_b) {
    const int rc = check_mlp(M, K, F, MOTIF_GATE_SILU, dtype);
    if (rc) return rc;
    Arena ws = {nullptr, 0};
    backward_of(ws, x, x_rs, w_gate, w_up, M, K, F, dtype, need_x, need_w, need_b);
    return ws.used;
}

extern "C" int motif_gated_mlp_bwd(const void* x, long x_rs, const void* w_gate, const void* w_up, const float* G, const float* U, const void* dh, long dh_rs,
                                   void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, void* workspace, long M, long K, long F, int act, int dtype, void* stream) {
    const int rc = check_mlp(M, K, F, act, dtype);
    if (rc) return rc;
    const bool need_x = dx, need_w = dw_gate || dw_up, need_b = db_gate || db_up;
    if (need_w && (!dw_gate || !dw_up)) return MOTIF_EINVAL;
    if (M < 1 || !x || !w_gate || !w_up || !G || !U || !dh || x_rs < 0 || dh_rs < 0 || !(need_x || need_w || need_b)) return MOTIF_EINVAL;
    if (!seq_aligned(G, 16) || !seq_aligned(U, 16)) return MOTIF_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    Arena ws = {(char*)workspace, 0};
    const Backward b = backward_of(ws, x, x_rs, w_gate, w_up, M, K, F, dtype, need_x, need_w, need_b);
    if (ws.used && !workspace) return MOTIF_EINVAL;
    if (b.one_pass) {
        const int grid = narrow_groups(M, F), slots = grid * (8 / column_runs(F));
        seq_dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (K <= 32) narrow_bwd<T, 2>(grid, x, x_rs, w_gate, w_up, dh, dh_rs, G, U, dx, b.dw_part, b.bias_part, b.peaks, (int)M, (int)K, (int)F, act, s);
            else narrow_bwd<T, 4>(grid, x, x_rs, w_gate, w_up, dh, dh_rs, G, U, dx, b.dw_part, b.bias_part, b.peaks, (int)M, (int)K, (int)F, act, s);
        });
        MOTIF_LAUNCH_CHECK();
        const int r = need_w ? seq_colsum2(b.dw_part, slots, F * K, dw_gate, dw_up, dtype, s) : MOTIF_OK;
        return r || !need_b ? r : seq_colsum2(b.bias_part, slots, F, db_gate, db_up, dtype, s);
    }
    lay_out(b.in, need_w, need_x, x, x_rs, w_gate, w_up, M, K, F, dtype, s);
    seq_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int rows = grad_rows(M, F);
        const int blocks = grad_blocks(M, F);
        auto launch = [&](auto* kernel, int grid) {
            kernel<<<grid, 256, 0, s>>>((const T*)dh, dh_rs, G, U, (int)M, (int)F, b.dg.ld, act, (void*)b.dg.p, b.dg.plane, b.dg.plane * b.dg.n, b.bias_part, rows, 4 * b.dg.plane * b.dg.n >= kSeqStream,
                                        b.peaks, blocks);
        };
        launch(gate_grad_kernel<T, false>, blocks);
        if constexpr (kRanged<T>) if (need_x || need_w) launch(gate_grad_kernel<T, true>, blocks < 256 ? blocks : 256);
    });
    if (need_b) {
        const int r = seq_colsum2(b.bias_part, cdiv(M, grad_rows(M, F)), F, db_gate, db_up, dtype, s);
        if (r) return r;
    }
    if (need_x) {                                        // the second pair continues the reduction of the first
        GemmArgs g = {};
        segments(g, b.dg, b.in.wg, b.in.wg);
        segments(g, b.du, b.in.wu, b.in.wu);
        g.lda = b.dg.ld; g.ldb = b.in.wg.ld;
        g.ka = b.dg.ld; g.kb = (int)F;
        g.units = units_of(b.dg.ld);
        g.M = (int)M; g.N = (int)K; g.wb = up8(K);
        g.c0 = dx; g.dtype = dtype;
        g.up = b.peaks ? b.peaks + grad_blocks(M, F) : nullptr;
        g.part = b.part;
        gemm_dtype<ONE>(dtype, b.dx, g, s);
    }
    if (need_w) {
        GemmArgs g = {};
        segments(g, b.in.x, b.dg, b.du);
        g.lda = b.in.x.ld; g.ldb = b.dg.ld;
        g.ka = g.kb = (int)M;
        g.units = units_of(M);
        g.M = (int)K; g.N = (int)F; g.wa = up8(K); g.wb = b.dg.ld;
        g.c0 = dw_gate; g.c1 = dw_up; g.dtype = dtype;
        g.up = b.peaks ? b.peaks + grad_blocks(M, F) : nullptr;
        g.part = b.part;
        gemm_dtype<TWO>(dtype, b.dw, g, s);
    }
    MOTIF_LAUNCH_CHECK();
    return MOTIF_OK;
}

extern "C" int motif_gated_mlp_tile(const void* x, long x_rs, const void* w_gate, const void* w_up, long M, long K, long F, int dtype, int product) {
    const int rc = check_mlp(M, K, F, MOTIF_GATE_SILU, dtype);
    if (rc || product < 0 || product > 3) return rc ? rc : MOTIF_EINVAL;
    if (product < 2) {
        Arena ws = {nullptr, 0};
        const Inputs f = inputs_of(ws, x, x_rs, w_gate, w_up, M, K, F, dtype);
        if ((M > kFewRows && narrow(K, F)) || few(M, K, F, dtype, f.lay_x || f.lay_w)) return 0;
        return fwd_plan(M, K, F, dtype, product == 1).big ? 256 : 128;
    }
    if (narrow_bwd(K, F)) return 0;
    return (product == 2 ? dx_plan(M, K, F, dtype) : dw_plan(M, K, F, dtype)).big ? 256 : 128;
}
