// gated_linear.hip -- the gated projection of a feed-forward block on pixel-major maps, and its backward pass:
//
//     g = x Wg^T + bg,  u = x Wu^T + bu,  z = act(g) * u            x [M][K], Wg, Wu [F][K], z [M][F]
//
// Forward: one product whose weight rows alternate 16 of Wg with 16 of Wu, so that a lane's accumulators hold g and u of the same
// elements and the activation and the product happen in registers: g and u never reach memory.
// Backward, 16-bit maps: the same product again, with dz in the epilogue: dg = dz u act'(g) and du = dz act(g), side by side in one map
// D [M][2 Fp] (Fp = F rounded up to 32, the columns between zero), with the bias gradients' partial sums in f32 beside the rounding to
// the map's type (a cotangent beyond f16's range becomes infinite there, as in every block that stores one).  Keeping g and u instead would round
// them to 16 bits, and at K = 256 their traffic costs about what the product does (34656 x 256 -> 1024: 142 MB written and 213 read, 57 us at the 6.2 TB/s of
// a large streaming pass, against 62).  f32 maps keep them: nothing is rounded, and the product costs five times as much as an elementwise pass
// (2280 x 512 -> 1365: 73 us against 14).
// Then dx = D [Wg; Wu] and [dWg; dWu] = D^T x, the latter split over the pixels and joined in a fixed order.
#include "common.h"

namespace {

constexpr int NT = 256;

enum { FWD, BWD, DX, DW };

struct GLArgs {
    const void *x, *wg, *wu, *dz;
    const float *bg, *bu;
    void *z, *D, *dx;
    float *pre;                      // f32 maps: g and u, [M][2 Fp], written by the forward pass for the backward one (or null)
    float *partial;                  // BWD: bias sums [row block][2 Fp];  DW: [split][2 Fp][K];  DX: [split][M][K], or null: dx is written
    int64_t M;
    int K, Kv, F, Fp, ldx, ldwg, ldwu, lddz, act;   // Kv: K in whole 16-byte vectors (what lies between is zero)
    int64_t split_rows;              // contraction per split: pixels (DW), columns of D (DX)
};

// ---- activation of the gate and its derivative ---------------------------------------------------------------------------------
// exp through v_exp_f32 and 1 / (1 + e) through v_rcp_f32 (about 1 ulp each, saturating: e = inf gives 0).  exp's argument is rounded before it: the
// result is off by about |g| half steps of f32 (SiLU at g = -20: 20 of them, 1.2e-6), GELU's exp(-g^2 / 2) by g^2 / 2.
// GELU's phi(g) = erfc(-g / sqrt 2) / 2.  16-bit maps: t P(t) exp(-g^2 / 2) for g < 0, 1 - that of -g otherwise, t = 1 / (1 + 0.545 |g| / sqrt 2),
// which shares its exp with the derivative.  t P(t) = exp(y^2) erfc(y) / 2 at y = |g| / sqrt 2 is smooth in t down to t = 0 (its limit is 1 / (2 y sqrt pi)), so
// a polynomial of degree 6, fitted for the smallest relative error over all t in (0, 1], has one of 4.3e-6 however far out the gate lies; with the
// exponential's 1.1e-5 down to g = -13, where exp(-g^2 / 2) leaves f32's normal range.  Half a step of f16 is 4.9e-4, of bf16 3.9e-3.  f32 maps take erfcf.
__device__ __forceinline__ float fast_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.4426950408889634f); }
template <int ACT, bool F32> __device__ __forceinline__ void gate_act(float g, float &a, float &da) {
    if constexpr (ACT == RDFC_ACT_RELU) {
        a = g > 0.f ? g : (g != g ? g : 0.f);
        da = g > 0.f ? 1.f : 0.f;
    } else if constexpr (ACT == RDFC_GATE_GELU) {
        const float e = fast_exp(-0.5f * g * g);
        float phi;
        if constexpr (F32) {
            phi = 0.5f * erfcf(g * -0.70710678118654752f);
        } else {
            const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.545f * 0.70710678118654752f, 1.f));
            float q = fmaf(0.0483367644f, t, -0.151893944f);
            q = fmaf(q, t, 0.0956667794f);
            q = fmaf(q, t, 0.0674590369f);
            q = fmaf(q, t, 0.133040484f);
            q = fmaf(q, t, 0.15364804f);
            q = fmaf(q, t, 0.153742316f);
            q *= t * e;
            phi = g < 0.f ? q : 1.f - q;
        }
        a = g * phi;
        da = fmaf(g * 0.39894228040143268f, e, phi);
    } else {
        const float s = __builtin_amdgcn_rcpf(1.f + fast_exp(-g));
        a = ACT == RDFC_ACT_SIGMOID ? s : g * s;
        da = ACT == RDFC_ACT_SIGMOID ? s * (1.f - s) : s * fmaf(g, 1.f - s, 1.f);
    }
}
// body(ACT as a type), chosen once per workgroup
template <typename F> __device__ __forceinline__ void with_gate(int act, F &&body) {
    if (act == RDFC_ACT_RELU) body(std::integral_constant<int, RDFC_ACT_RELU>{});
    else if (act == RDFC_GATE_GELU) body(std::integral_constant<int, RDFC_GATE_GELU>{});
    else if (act == RDFC_ACT_SIGMOID) body(std::integral_constant<int, RDFC_ACT_SIGMOID>{});
    else body(std::integral_constant<int, RDFC_GATE_SILU>{});
}

// sum over the 16 lanes of a row of lanes
__device__ __forceinline__ float row16_sum(float v) {
    auto add = [&](auto ctrl) { v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true)); };
    add(std::integral_constant<int, 0xB1>{});
    add(std::integral_constant<int, 0x4E>{});
    add(std::integral_constant<int, 0x141>{});
    add(std::integral_constant<int, 0x140>{});
    return v;
}

// Rows that are not whole aligned vectors (an odd channel count, an odd slice) are copied to dense rows of Kv = K rounded up to whole
// 16-byte vectors first, zeros behind K: one pass over an operand that the product reads many times.  blockIdx.y: operand.
template <typename T> __global__ __launch_bounds__(NT) void gated_pack_kernel(const T *__restrict__ s0, const T *__restrict__ s1, T *__restrict__ d0, T *__restrict__ d1,
                                                                              int64_t rows, int K, int Kv, int ld0, int ld1) {
    constexpr int VEC = Elem<T>::VEC;
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    const int per = Kv / VEC;
    if (i >= rows * per) return;
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * VEC;
    const T *src = blockIdx.y ? s1 + r * ld1 : s0 + r * ld0;
    Vec16<T> v;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v.set(k, c + k < K ? Elem<T>::ld(src + c + k) : 0.f);
    v.store((blockIdx.y ? d1 : d0) + r * Kv + c);
}

// ---- the tiled kernel --------------------------------------------------------------------------------------------------------------
// Four waves, each WTP x WTQ of a (2 WTP) x (2 WTQ) tile; operands go global -> LDS by LDS-DMA (buffer_load ... lds) into a ring of three
// K-steps of 64 bytes a row, filled two steps ahead; one raw barrier and one counted wait per step.  A 64 x 64 wave tile needs 48 KB of LDS and
// 107 registers: three workgroups share a CU, and one's prologue and epilogue run under the others' MFMAs.  That matters more here than a
// cheaper K loop: at K = 256 half of the forward pass's time is not the K loop (one K-step instead of eight: 33 of 64 us).
//
// Measured (16-bit, launches in a row): forward 34656 x 256 -> 1024 62 us, 588 TFLOP/s (a library product of the same size without activation: 72 us);
// 8816 x 512 -> 2048 with GELU 54 to 56 us (library 76); 34656 x 1024 -> 1024 160 us, 908 TFLOP/s (library 151), where the matrix pipes are busy for
// half of the cycles.  The first forward + backward: 262 us.  Its launches in a kernel trace, where none overlap (best of 20, the means are up to a sixth
// longer): forward 65, D 96 (6 % more with dz read eight bytes a lane in the epilogue), dx 58, dW 46, the joins 6 and 5 us.
// Tried and not kept: fragments read a step ahead in a second register set (no change), steps of 128 bytes in two pairs of slots (two
// workgroups a CU: 60 -> 70 us at K = 256), eight waves on 256 x 128 with a ring of three 128-byte steps (75 us at K = 256, 174 at K = 1024).
//
// An operand whose contraction index is contiguous in memory (ROW) has an LDS image [row][64 bytes], the 16-byte chunk c of row r at c ^ (r >> 1 & 3):
// eight lanes of a fragment read (rows r .. r + 7, one chunk) then cover all 128 bytes of the banks.  One whose contraction index is the
// row index (COL: the weights in dx, x and D in dW) has the image [k][columns], read transposed (ds_read_b64_tr_b16; plain
// dwords in f32), its 32-byte pairs (64-byte units in f32) permuted by the row for the same reason.  Rows and columns that do not exist
// are beyond the descriptor's extent and arrive as zeros, or end in accumulators that are never stored; a K tail is masked per lane.
constexpr unsigned DEAD = 0x80000000u;
__device__ __forceinline__ void bdma16(unsigned voff, u32x4 rsrc, unsigned soff, unsigned lds_base) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ u32x4 make_rsrc(const void *base, int64_t bytes) {
    const unsigned long long b = reinterpret_cast<unsigned long long>(base);
    bytes = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((unsigned)b);
    r[1] = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32) & 0xffffu);
    r[2] = __builtin_amdgcn_readfirstlane((unsigned)bytes);
    r[3] = 0x00020000u;
    return r;
}

// one operand of W rows (tile extent): DMA pieces of 1 KB, piece i of the step's image
template <int ES, bool COL, int W> struct Image {
    static constexpr int ROWB = COL ? W * ES : 64;               // bytes per image row
    static constexpr int PIECES = W * 64 / 1024;
    static __device__ int row(int i, int lane) { return (i * 1024 + lane * 16) / ROWB; }
    static __device__ int swz(int row) {
        if (!COL) return (row >> 1) & 3;                         // 16-byte chunks
        if (ES == 4) return (row >> 2) & 3;                      // 64-byte units
        return ROWB == 128 ? (row & 3) : (row & 3) | ((row >> 3) & 1) << 2;      // 32-byte pairs
    }
    // byte offset, within the source row's window, of what lane's 16 bytes of piece i hold
    static __device__ unsigned src(int i, int lane) {
        const int r = row(i, lane), slot = (i * 64 + lane) % (ROWB / 16), s = swz(r);
        if (!COL) return (unsigned)(slot ^ s) * 16;
        if (ES == 4) return (unsigned)(slot ^ s << 2) * 16;
        return (unsigned)(slot ^ s << 1) * 16;
    }
};

template <int DT, int MODE, int WTP, int WTQ>
__global__ __launch_bounds__(NT, 2) void gated_dma_kernel(GLArgs p, int tiles_p, int64_t tiles_q) {
    using T = typename std::conditional<DT == RDFC_F32, float, typename std::conditional<DT == RDFC_F16, f16_t, bf16_t>::type>::type;
    constexpr int ES = DT == RDFC_F32 ? 4 : 2, BKE = 64 / ES, BP = 2 * WTP, BQ = 2 * WTQ, RING = 3, LOOK = 2;
    constexpr bool PCOL = MODE == DX || MODE == DW, QCOL = MODE == DW, GATED = MODE == FWD || MODE == BWD;
    using IP = Image<ES, PCOL, BP>;
    using IQ = Image<ES, QCOL, BQ>;
    constexpr int PB = BP * 64, SLOT = PB + BQ * 64, NP = IP::PIECES / 4, NQ = IQ::PIECES / 4;
    constexpr int MT = WTP / 16, QT = WTQ / 16;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wp = wave >> 1, wq = wave & 1;
    // Workgroups are dealt to the 8 XCDs in turn.  Each XCD takes one eighth of the tiles, P tiles of a Q tile (the pixels) side by side: they
    // share what its L2 holds of the pixels, and every XCD has the same number of them whatever the sizes.
    const int64_t tiles = tiles_q * tiles_p, per = (tiles + 7) >> 3, local = blockIdx.x >> 3, index = (blockIdx.x & 7) * per + local;
    if (local >= per || index >= tiles) return;
    int64_t tq = index / tiles_p;
    int tp = (int)(index - tq * tiles_p);
    int64_t kbeg = 0, kend = MODE == DX ? 2 * p.Fp : p.Kv;
    int split = 0;
    if constexpr (MODE == DX) {
        // (the splits of a tile side by side)
        const int splits = (int)((kend + p.split_rows - 1) / p.split_rows);
        split = tp % splits;
        tp /= splits;
        kbeg = split * p.split_rows;
        kend = min(kbeg + p.split_rows, kend);
    }
    int64_t q0 = tq * BQ;
    if constexpr (MODE == DW) {
        // (the pixels are contracted: tq numbers the splits, tp the output tiles)
        kbeg = tq * p.split_rows;
        kend = min(kbeg + p.split_rows, p.M);
        const int nq = (2 * p.Fp + BQ - 1) / BQ;
        q0 = (int64_t)(tp % nq) * BQ;
        tp /= nq;
    }
    const int p0 = tp * (GATED ? BP / 2 : BP);
    const int G = (int)((kend - kbeg + BKE - 1) / BKE);

    // ---- sources: per-lane offsets within a step, wave-uniform descriptors -----------------------------------------------------------
    const T *x = (const T *)p.x, *wg = (const T *)p.wg, *wu = (const T *)p.wu, *D = (const T *)p.D;
    unsigned offp[NP], offq[NQ];
    u32x4 rp[2], rq;
    if constexpr (GATED) {
        rp[0] = make_rsrc(wg + (int64_t)p0 * p.ldwg, ((int64_t)(p.F - p0 - 1) * p.ldwg + p.Kv) * ES);
        rp[1] = make_rsrc(wu + (int64_t)p0 * p.ldwu, ((int64_t)(p.F - p0 - 1) * p.ldwu + p.Kv) * ES);
        rq = make_rsrc(x + q0 * p.ldx, ((p.M - q0 - 1) * p.ldx + p.Kv) * ES);
    } else if constexpr (MODE == DX) {
        rq = make_rsrc(D + q0 * 2 * p.Fp, (p.M - q0) * 2 * p.Fp * ES);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int i = k * 4 + wave, r = IP::row(i, lane);
        // (GATED: piece i holds 16 rows of one kind, i & 1, of the features 16 (i >> 1) ..)
        if constexpr (GATED) offp[k] = (unsigned)((i >> 1) * 16 + (r & 15)) * (unsigned)((i & 1 ? p.ldwu : p.ldwg) * ES) + IP::src(i, lane);
        else offp[k] = (unsigned)r * (unsigned)((MODE == DX ? p.ldwg : p.ldx) * ES) + IP::src(i, lane);
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
        const int i = k * 4 + wave;
        offq[k] = (unsigned)IQ::row(i, lane) * (unsigned)((GATED ? p.ldx : 2 * p.Fp) * ES) + IQ::src(i, lane);
    }
    auto issue = [&](int h, int slot) {
        const bool live = h < G;
        const unsigned base = lds0 + slot * SLOT;
        const int64_t k0 = kbeg + (int64_t)h * BKE;
        u32x4 r0 = rp[0], r1 = rp[1], rq_ = rq;
        unsigned so = (unsigned)(k0 * ES);
        if constexpr (MODE == DX) {
            const bool up = k0 >= p.Fp;                          // (Fp is a multiple of the step: a step lies in one half)
            const int64_t f = up ? k0 - p.Fp : k0;
            const int ld = up ? p.ldwu : p.ldwg;
            r0 = make_rsrc((up ? wu : wg) + f * ld + p0, live ? ((int64_t)(p.F - f - 1) * ld + p.Kv - p0) * ES : 0);
        } else if constexpr (MODE == DW) {
            r0 = make_rsrc(x + k0 * p.ldx + p0, live ? ((kend - k0 - 1) * p.ldx + p.Kv - p0) * ES : 0);
            rq_ = make_rsrc(D + k0 * 2 * p.Fp + q0, live ? ((kend - k0) * 2 * p.Fp - q0) * ES : 0);
            so = 0;
        }
        if constexpr (GATED) {
            if (!live) r0[2] = r1[2] = rq_[2] = 0;
        }
        if constexpr (MODE == DX) {
            if (!live) rq_[2] = 0;
        }
        // a K tail: chunks at or behind kend are zero in the ROW images
        const bool tail = k0 + BKE > kend;
        auto off = [&](unsigned o, int i, bool col, unsigned src) { return !col && tail && k0 + (int)(src / ES) >= kend ? DEAD : o; };
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const int i = k * 4 + wave;
            bdma16(off(offp[k], i, PCOL, PCOL ? 0 : IP::src(i, lane)), GATED && (wave & 1) ? r1 : r0, PCOL ? 0 : so, base + i * 1024);
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
            const int i = k * 4 + wave;
            bdma16(off(offq[k], i, QCOL, QCOL ? 0 : IQ::src(i, lane)), rq_, QCOL ? 0 : so, base + PB + i * 1024);
        }
    };

    // (GATED: rows alternate 16 features of the gate with 16 of the other projection, and the accumulators start at the biases)
    f32x4 acc[MT][QT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        f32x4 first = {0, 0, 0, 0};
        if constexpr (GATED) {
            const float *bias = i & 1 ? p.bu : p.bg;
            const int f = p0 + wp * (WTP / 2) + 16 * (i >> 1) + 4 * (lane >> 4);
            if (bias != nullptr) {
#pragma unroll
                for (int r = 0; r < 4; ++r) first[r] = f + r < p.F ? bias[f + r] : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < QT; ++j) acc[i][j] = first;
    }

    // ---- fragments: 16 rows (or columns) from `first`, the step's whole contraction range ---------------------------------------------
    const int l16 = lane & 15, g4 = lane >> 4;
    auto frag16 = [&](const unsigned char *S, auto image, bool col, int first) -> bf16x8 {
        using IM = decltype(image);
        if (!col) {
            const int r = first + l16;
            return *reinterpret_cast<const bf16x8 *>(S + r * 64 + ((g4 ^ ((r >> 1) & 3)) << 4));
        }
        const int r0 = 8 * g4 + (l16 >> 2);
        const unsigned char *a = S + r0 * IM::ROWB + (((first >> 4) ^ IM::swz(r0)) << 5) + (l16 & 3) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)a);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a + 4 * IM::ROWB));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        return __builtin_bit_cast(bf16x8, u32x4{l2[0], l2[1], h2[0], h2[1]});
    };
    auto frag32 = [&](const unsigned char *S, auto image, bool col, int first) -> f32x4 {
        using IM = decltype(image);
        if (!col) {
            const int r = first + l16;
            return *reinterpret_cast<const f32x4 *>(S + r * 64 + ((g4 ^ ((r >> 1) & 3)) << 4));
        }
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = 4 * g4 + k;
            v[k] = *reinterpret_cast<const float *>(S + r * IM::ROWB + (((first >> 4) ^ IM::swz(r)) << 6) + l16 * 4);
        }
        return v;
    };

    // BWD: dz of 16 pixels at a time in whole rows, one 16-byte load a lane; the first ones under the K loop
    constexpr int DCH = WTP / 16, DROW = WTP + 16;               // 16-byte chunks of the wave's features in a pixel, bytes of its staging row
    auto fetch_dz = [&](int j) {
        u32x4 v = {0, 0, 0, 0};
        const int64_t m = q0 + wq * WTQ + 16 * j + lane / DCH;
        const int f = p0 + wp * (WTP / 2) + lane % DCH * 8;
        if (lane < 16 * DCH && m < p.M && f < p.F) {
            const bf16_t *src = reinterpret_cast<const bf16_t *>(p.dz) + m * p.lddz + f;
            if (p.lddz % 8 == 0 && (reinterpret_cast<size_t>(p.dz) & 15) == 0 && f + 8 <= p.F) {
                v = *reinterpret_cast<const u32x4 *>(src);
            } else {
                bf16x8 e = __builtin_bit_cast(bf16x8, v);
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (f + r < p.F) e[r] = src[r];
                v = __builtin_bit_cast(u32x4, e);
            }
        }
        return v;
    };
    u32x4 next_dz;
    if constexpr (MODE == BWD) next_dz = fetch_dz(0);

#pragma unroll
    for (int h = 0; h < LOOK; ++h) issue(h, h);
    int slot = 0, fill = LOOK;
    for (int g = 0; g < G; ++g) {
        wait_vm_and_reads<(LOOK - 1) * (NP + NQ)>();
        __builtin_amdgcn_s_barrier();
        issue(g + LOOK, fill);                                   // (its slot was last read in step g - 1: every wave is past the barrier)
        const unsigned char *S = smem + slot * SLOT;
        slot = slot == RING - 1 ? 0 : slot + 1;
        fill = fill == RING - 1 ? 0 : fill + 1;
        if constexpr (ES == 2) {
            bf16x8 a[MT], b[QT];
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = frag16(S, IP{}, PCOL, wp * WTP + 16 * i);
#pragma unroll
            for (int j = 0; j < QT; ++j) b[j] = frag16(S + PB, IQ{}, QCOL, wq * WTQ + 16 * j);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < QT; ++j) acc[i][j] = mma16<DT>(a[i], b[j], acc[i][j]);
        } else {
            f32x4 a[MT], b[QT];
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = frag32(S, IP{}, PCOL, wp * WTP + 16 * i);
#pragma unroll
            for (int j = 0; j < QT; ++j) b[j] = frag32(S + PB, IQ{}, QCOL, wq * WTQ + 16 * j);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < QT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][k], b[j][k], acc[i][j], 0, 0, 0);
        }
    }
    wait_vm_and_reads<0>();
    __syncthreads();                                             // every wave is done with the ring: it becomes the staging tiles

    // ---- epilogue: 16 pixels at a time through the wave's staging tile, then whole rows ---------------------------------------------
    const int q4 = g4 * 4;
    constexpr int OW = GATED ? WTP / 2 : WTP;                    // output channels of the wave
    constexpr int OROW = OW * ES + 16;
    static_assert(4 * 16 * OROW <= RING * SLOT, "the staging tiles live in the ring");
    unsigned char *Ot = smem + wave * 16 * OROW;
    auto put = [&](int ch, const float (&v)[4]) {                // channels ch .. ch + 3 of the lane's pixel
        if constexpr (ES == 4) {
            *reinterpret_cast<f32x4 *>(Ot + l16 * OROW + ch * 4) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            bf16x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = cvt16<DT>(v[r]);
            *reinterpret_cast<bf16x4 *>(Ot + l16 * OROW + ch * 2) = o;
        }
    };
    // rows m .. m + 15 of out (row stride ld, `nch` of the wave's channels exist)
    auto flush = [&](T *out, int64_t m, int ld, int nch, bool vec) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        constexpr int CH = OW * ES / 16, VE = 16 / ES;           // 16-byte chunks per row, elements per chunk
#pragma unroll
        for (int e = lane; e < 16 * CH; e += 64) {
            const int row = e / CH, c = e % CH;
            if (m + row >= p.M || c * VE >= nch) continue;
            const unsigned char *src = Ot + row * OROW + c * 16;
            T *dst = out + (m + row) * ld + c * VE;
            if (vec && c * VE + VE <= nch) *reinterpret_cast<u32x4 *>(dst) = *reinterpret_cast<const u32x4 *>(src);
            else
                for (int r = 0; r < VE && c * VE + r < nch; ++r) dst[r] = reinterpret_cast<const T *>(src)[r];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    if constexpr (GATED) {
        const int fw = p0 + wp * OW;                             // the wave's first feature
        with_gate(p.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if constexpr (MODE == FWD) {
                const bool vec = p.F * ES % 16 == 0 && (reinterpret_cast<size_t>(p.z) & 15) == 0;
#pragma unroll
                for (int j = 0; j < QT; ++j) {
                    if constexpr (ES == 4) {
                        if (p.pre != nullptr) {
#pragma unroll
                            for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
                                for (int i = 0; i < MT / 2; ++i) {
                                    const float v[4] = {acc[2 * i + kind][j][0], acc[2 * i + kind][j][1], acc[2 * i + kind][j][2], acc[2 * i + kind][j][3]};
                                    put(16 * i + q4, v);
                                }
                                flush(p.pre + kind * p.Fp + fw, q0 + wq * WTQ + 16 * j, 2 * p.Fp, p.Fp - fw, true);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MT / 2; ++i) {
                        float v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float a, da;
                            gate_act<ACT, ES == 4>(acc[2 * i][j][r], a, da);
                            v[r] = a * acc[2 * i + 1][j][r];
                        }
                        put(16 * i + q4, v);
                    }
                    flush((T *)p.z + fw, q0 + wq * WTQ + 16 * j, p.F, p.F - fw, vec);
                }
            } else {
                float sg[MT / 2][4], su[MT / 2][4];
#pragma unroll
                for (int i = 0; i < MT / 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sg[i][r] = su[i][r] = 0.f;
                static_assert(16 * DCH <= 64 && 4 * 16 * (OROW + DROW) <= RING * SLOT, "one load a lane; both staging tiles live in the ring");
                unsigned char *Dt = smem + 4 * 16 * OROW + wave * 16 * DROW;
#pragma unroll
                for (int j = 0; j < QT; ++j) {
                    const int64_t m = q0 + wq * WTQ + 16 * j + l16;
                    if (lane < 16 * DCH) *reinterpret_cast<u32x4 *>(Dt + lane / DCH * DROW + lane % DCH * 16) = next_dz;
                    if (j + 1 < QT) next_dz = fetch_dz(j + 1);
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    float w[MT / 2][4];
#pragma unroll
                    for (int i = 0; i < MT / 2; ++i) {
                        const int f = fw + 16 * i + q4;
                        const bf16x4 t = *reinterpret_cast<const bf16x4 *>(Dt + l16 * DROW + (16 * i + q4) * 2);
                        float dz[4], v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) dz[r] = f32of<DT>(t[r]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float a, da;
                            gate_act<ACT, ES == 4>(acc[2 * i][j][r], a, da);
                            // (a pixel or feature that is not there: zero, whatever its accumulators hold)
                            const bool on = m < p.M && f + r < p.F;
                            v[r] = on ? dz[r] * acc[2 * i + 1][j][r] * da : 0.f;
                            w[i][r] = on ? dz[r] * a : 0.f;
                            sg[i][r] += v[r];
                            su[i][r] += w[i][r];
                        }
                        put(16 * i + q4, v);
                    }
                    flush((T *)p.D + fw, q0 + wq * WTQ + 16 * j, 2 * p.Fp, p.Fp - fw, true);
#pragma unroll
                    for (int i = 0; i < MT / 2; ++i) put(16 * i + q4, w[i]);
                    flush((T *)p.D + p.Fp + fw, q0 + wq * WTQ + 16 * j, 2 * p.Fp, p.Fp - fw, true);
                }
                if (p.partial == nullptr) return;
                __syncthreads();
                float *bsum = reinterpret_cast<float *>(smem);   // [wq][kind][BP / 2]
#pragma unroll
                for (int i = 0; i < MT / 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float a = row16_sum(sg[i][r]), b = row16_sum(su[i][r]);
                        if (l16 == 0) {
                            bsum[wq * BP + wp * OW + 16 * i + q4 + r] = a;
                            bsum[wq * BP + BP / 2 + wp * OW + 16 * i + q4 + r] = b;
                        }
                    }
                __syncthreads();
                for (int e = tid; e < BP; e += NT) {
                    const int f = p0 + e % (BP / 2), kind = e / (BP / 2);
                    if (f < p.Fp) p.partial[(size_t)tq * 2 * p.Fp + kind * p.Fp + f] = bsum[e] + bsum[BP + e];
                }
            }
        });
    } else if constexpr (MODE == DX) {
        const int kw = p0 + wp * WTP;
        if (p.partial != nullptr) {
#pragma unroll
            for (int j = 0; j < QT; ++j) {
                const int64_t m = q0 + wq * WTQ + 16 * j + l16;
                if (m >= p.M) continue;
                float *out = p.partial + ((size_t)split * p.M + m) * p.K;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    for (int r = 0; r < 4; ++r)
                        if (kw + 16 * i + q4 + r < p.K) out[kw + 16 * i + q4 + r] = acc[i][j][r];
            }
            return;
        }
        const bool vec = p.K * ES % 16 == 0 && (reinterpret_cast<size_t>(p.dx) & 15) == 0;
#pragma unroll
        for (int j = 0; j < QT; ++j) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                put(16 * i + q4, v);
            }
            flush((T *)p.dx + kw, q0 + wq * WTQ + 16 * j, p.K, p.K - kw, vec);
        }
    } else {
#pragma unroll
        for (int j = 0; j < QT; ++j) {
            const int64_t q = q0 + wq * WTQ + 16 * j + l16;
            if (q >= 2 * p.Fp) continue;
            float *out = p.partial + ((size_t)tq * 2 * p.Fp + q) * p.K;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int kk = p0 + wp * WTP + 16 * i + q4;
                if ((p.K & 3) == 0) {
                    if (kk < p.K) *reinterpret_cast<f32x4 *>(out + kk) = acc[i][j];
                } else {
                    for (int r = 0; r < 4; ++r)
                        if (kk + r < p.K) out[kk + r] = acc[i][j][r];
                }
            }
        }
    }
}

// D and the bias sums of ACT_ROWS pixels from the kept g and u (f32): 64 lanes of 4 features x 4 row lanes
constexpr int ACT_ROWS = 64;
__global__ __launch_bounds__(NT) void gated_act_kernel(GLArgs p) {
    __shared__ float red[4][2][256];
    const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6, f = (blockIdx.y * 64 + cl) * 4;
    const int64_t m0 = (int64_t)blockIdx.x * ACT_ROWS, m1 = min(m0 + ACT_ROWS, p.M);
    float sg[4] = {0.f, 0.f, 0.f, 0.f}, su[4] = {0.f, 0.f, 0.f, 0.f};
    const bool vec = p.lddz % 4 == 0 && (reinterpret_cast<size_t>(p.dz) & 15) == 0;
    if (f < p.Fp) {
        with_gate(p.act, [&](auto act) {
#pragma unroll 4
            for (int64_t m = m0 + rl; m < m1; m += 4) {
                const f32x4 g = *reinterpret_cast<const f32x4 *>(p.pre + m * 2 * p.Fp + f), u = *reinterpret_cast<const f32x4 *>(p.pre + m * 2 * p.Fp + p.Fp + f);
                const float *src = (const float *)p.dz + m * p.lddz + f;
                f32x4 dz = {0.f, 0.f, 0.f, 0.f}, dg, du;
                if (vec && f + 3 < p.F) dz = *reinterpret_cast<const f32x4 *>(src);
                else
                    for (int r = 0; r < 4; ++r)
                        if (f + r < p.F) dz[r] = src[r];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float a, da;
                    gate_act<decltype(act)::value, true>(g[r], a, da);
                    dg[r] = f + r < p.F ? dz[r] * u[r] * da : 0.f;
                    du[r] = f + r < p.F ? dz[r] * a : 0.f;
                    sg[r] += dg[r];
                    su[r] += du[r];
                }
                *reinterpret_cast<f32x4 *>((float *)p.D + m * 2 * p.Fp + f) = dg;
                *reinterpret_cast<f32x4 *>((float *)p.D + m * 2 * p.Fp + p.Fp + f) = du;
            }
        });
    }
    if (p.partial == nullptr) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        red[rl][0][cl * 4 + r] = sg[r];
        red[rl][1][cl * 4 + r] = su[r];
    }
    __syncthreads();
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= p.Fp) return;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        p.partial[(size_t)blockIdx.x * 2 * p.Fp + k * p.Fp + c] = (red[0][k][threadIdx.x] + red[1][k][threadIdx.x]) + (red[2][k][threadIdx.x] + red[3][k][threadIdx.x]);
}

// o0 (o1: the second half of a part) [n] = sum over the parts of partial[part][step], in the order of the parts, in f64.  V elements a thread
template <typename TO, int V> __global__ __launch_bounds__(NT) void gated_join_kernel(const float *__restrict__ partial, int parts, size_t n, size_t step, TO *o0, TO *o1) {
    const size_t i = ((size_t)blockIdx.x * NT + threadIdx.x) * V;
    TO *o = blockIdx.y ? o1 : o0;
    if (i >= n || o == nullptr) return;
    const float *src = partial + i + (blockIdx.y ? step / 2 : 0);
    double s[V] = {};
#pragma unroll 8
    for (int k = 0; k < parts; ++k) {
        if constexpr (V == 4) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(src + k * step);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] += (double)v[r];
        } else {
            s[0] += (double)src[k * step];
        }
    }
#pragma unroll
    for (int r = 0; r < V; ++r) Elem<TO>::st(o + i + r, (float)s[r]);
}
template <typename TO> void join(const float *partial, int parts, size_t n, size_t step, TO *o0, TO *o1, int halves, hipStream_t st) {
    if (n % 4 == 0 && step % 8 == 0) gated_join_kernel<TO, 4><<<dim3((unsigned)((n / 4 + NT - 1) / NT), halves), NT, 0, st>>>(partial, parts, n, step, o0, o1);
    else gated_join_kernel<TO, 1><<<dim3((unsigned)((n + NT - 1) / NT), halves), NT, 0, st>>>(partial, parts, n, step, o0, o1);
}

// out[kind][f] = sum over the row blocks of partial[block][kind * Fp + f]: 32 columns x 16 row lanes per workgroup
__global__ __launch_bounds__(512) void gated_bias_kernel(const float *__restrict__ partial, int blocks, int F, int Fp, float *__restrict__ o0, float *__restrict__ o1) {
    __shared__ double red[16][32];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;      // (2 Fp is a multiple of 64)
    double s = 0.;
#pragma unroll 8
    for (int k = rl; k < blocks; k += 16) s += (double)partial[(size_t)k * 2 * Fp + c];
    red[rl][cl] = s;
    __syncthreads();
    if (rl != 0) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][cl];
    const int kind = c >= Fp, f = kind ? c - Fp : c;
    float *o = kind ? o1 : o0;
    if (o != nullptr && f < F) o[f] = (float)s;
}

// what the kernel needs of an operand: rows of whole 16-byte vectors, and offsets of a tile that fit 31 bits
bool dma_ok(const void *p, int64_t ld, int dtype) {
    return (reinterpret_cast<size_t>(p) & 15) == 0 && ld % rdfc_vec(dtype) == 0 && ld <= (1 << 20);
}
size_t up256(size_t b) { return (b + 255) / 256 * 256; }
// dense copies of the operands that need one, at the start of the scratch memory
struct Packs {
    bool x, w;
    size_t x_bytes, w_bytes;                                     // w: of one of the two
    size_t bytes() const { return x_bytes + 2 * w_bytes; }
};
Packs packs_of(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu) {
    const int vec = rdfc_vec(d->dtype), es = 16 / vec;
    const size_t kv = (size_t)(d->K + vec - 1) / vec * vec;
    Packs q;
    q.x = d->K % vec != 0 || !dma_ok(x, d->ldx, d->dtype);
    q.w = d->K % vec != 0 || !dma_ok(wg, d->ldwg, d->dtype) || !dma_ok(wu, d->ldwu, d->dtype) || d->ldwg != d->ldwu;
    q.x_bytes = q.x ? up256((size_t)d->M * kv * es) : 0;
    q.w_bytes = q.w ? up256((size_t)d->F * kv * es) : 0;
    return q;
}
// the copies; p's operands become them
int pack(const rdfc_gated_desc *d, const Packs &q, GLArgs &p, void *scratch, hipStream_t st, const char *name) {
    const int vec = rdfc_vec(d->dtype), per = p.Kv / vec;
    unsigned char *at = (unsigned char *)scratch;
    auto run = [&](const void *s0, const void *s1, void *d0, void *d1, int64_t rows, int ld0, int ld1) -> int {
        const int64_t blocks = (rows * per + NT - 1) / NT;
        RDFC_REQUIRE(blocks < (1ll << 31), "%s: %lld rows are too many", name, (long long)rows);
        RDFC_DISPATCH(d->dtype, (gated_pack_kernel<T><<<dim3((unsigned)blocks, s1 ? 2 : 1), NT, 0, st>>>((const T *)s0, (const T *)s1, (T *)d0, (T *)d1, rows, p.K, p.Kv, ld0, ld1)));
        RDFC_LAUNCH_CHECK(name);
        return 0;
    };
    if (q.x) {
        if (run(p.x, nullptr, at, nullptr, d->M, p.ldx, 0)) return 2;
        p.x = at;
        p.ldx = p.Kv;
        at += q.x_bytes;
    }
    if (q.w) {
        if (run(p.wg, p.wu, at, at + q.w_bytes, d->F, p.ldwg, p.ldwu)) return 2;
        p.wg = at;
        p.wu = at + q.w_bytes;
        p.ldwg = p.ldwu = p.Kv;
    }
    return 0;
}

struct Tile {
    int wtp, wtq;
};
// Wave tile from the workgroups that 64 x 64 gives: below one per CU the chip is better filled by 32 x 32 (288 x 512 -> 1365, f16: 8.3 us against
// 11.3; f32 dx of 2280 x 512: 126 against 205).  128 x 64 moves a quarter fewer bytes through the L1 per product, but leaves two
// workgroups on a CU where 64 x 64 has three, and the backward kernel spills: it pays in the forward pass alone, from
// K = 768 (34656 x 1024 -> 1024, f16: 159 us against 179; at K = 256 63 against 60, at 512 56 against 56).
template <typename F> Tile tile_of(F &&of, bool wide = false) {
    if (wide && of(Tile{128, 64}) >= 384) return Tile{128, 64};
    return of(Tile{64, 64}) >= 256 ? Tile{64, 64} : Tile{32, 32};
}
template <int MODE> int launch_dma(const GLArgs &p, int dtype, Tile t, int tiles_p, int64_t tiles_q, hipStream_t st, const char *name) {
    const int64_t grid = (tiles_q * tiles_p + 7) / 8 * 8;
    RDFC_REQUIRE(grid < (1ll << 31), "%s: %lld workgroups are too many", name, (long long)grid);
    auto go = [&](auto dt, auto wtp, auto wtq) {
        constexpr int WTP = decltype(wtp)::value, WTQ = decltype(wtq)::value, LDS = 3 * (2 * WTP + 2 * WTQ) * 64;
        auto kernel = gated_dma_kernel<decltype(dt)::value, MODE, WTP, WTQ>;
        if (LDS > 65536) {
            static bool set[64] = {};                            // (per device; a race sets it twice)
            int dev = 0;
            if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
            if (!set[dev]) set[dev] = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) == hipSuccess;
        }
        kernel<<<dim3((unsigned)grid), NT, LDS, st>>>(p, tiles_p, tiles_q);
    };
    auto size = [&](auto dt) {
        if constexpr (MODE == FWD) {
            if (t.wtp == 128) {
                go(dt, std::integral_constant<int, 128>{}, std::integral_constant<int, 64>{});
                return;
            }
        }
        if (t.wtp == 64) go(dt, std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
        else go(dt, std::integral_constant<int, 32>{}, std::integral_constant<int, 32>{});
    };
    if (dtype == RDFC_BF16) size(std::integral_constant<int, RDFC_BF16>{});
    else if (dtype == RDFC_F16) size(std::integral_constant<int, RDFC_F16>{});
    else if constexpr (MODE != BWD) size(std::integral_constant<int, RDFC_F32>{});
    RDFC_LAUNCH_CHECK(name);
    return 0;
}

struct Plan {
    int Fp, row_blocks, splits, dx_splits;
    Tile gated, dx, dw;
    int64_t split_rows, dx_cols;
    size_t d_bytes, bias_floats, w_floats, dx_floats;
};
Plan plan_of(const rdfc_gated_desc *d) {
    Plan p;
    p.Fp = (d->F + 31) / 32 * 32;                                // (D's halves: whole K-steps of the product with the weights)
    p.gated = tile_of([&](Tile t) { return cdiv(p.Fp, t.wtp) * (int64_t)cdiv(d->M, 2 * t.wtq); });
    p.dx = tile_of([&](Tile t) { return cdiv(d->K, 2 * t.wtp) * (int64_t)cdiv(d->M, 2 * t.wtq); });
    p.row_blocks = cdiv(d->M, 64);                               // (of the smallest tile: an upper bound)
    // dx: the contraction (2 Fp) is split where its tiles would leave CUs idle, f32 parts joined afterwards (2280 x 512, f32: 126 -> 91 us)
    const int64_t dx_tiles = (int64_t)cdiv(d->K, 2 * p.dx.wtp) * cdiv(d->M, 2 * p.dx.wtq);
    int64_t ds = dx_tiles > 0 && p.dx.wtp == 32 ? 1024 / dx_tiles : 1;
    const int64_t ds_most = 2 * p.Fp / 256;
    ds = ds > 8 ? 8 : ds;
    ds = ds > ds_most ? ds_most : ds;
    ds = ds < 1 ? 1 : ds;
    p.dx_cols = (2 * p.Fp / ds + 31) / 32 * 32;
    p.dx_splits = (int)((2 * p.Fp + p.dx_cols - 1) / p.dx_cols);
    const int64_t most = (d->M + 255) / 256;
    p.dw = tile_of([&](Tile t) { return cdiv(d->K, 2 * t.wtp) * (int64_t)cdiv(2 * p.Fp, 2 * t.wtq) * (most < 32 ? most : 32); });
    const int64_t tiles = (int64_t)cdiv(d->K, 2 * p.dw.wtp) * cdiv(2 * p.Fp, 2 * p.dw.wtq);
    // two workgroups a CU (f32: three, what fits).  More parts cost the 16-bit maps more in the join than they fill: 34656 x 256 -> 1024, f16,
    // 512 / 768 workgroups: 60 / 69 us; f32 2280 x 512 -> 1365: 76 / 70
    int64_t s = (d->dtype == RDFC_F32 ? 768 : 512) / tiles;
    s = s > most ? most : s;
    s = s < 1 ? 1 : s;
    p.split_rows = ((d->M + s - 1) / s + 31) / 32 * 32;
    if (p.split_rows < 32) p.split_rows = 32;
    p.splits = (int)((d->M + p.split_rows - 1) / p.split_rows);
    p.d_bytes = ((size_t)d->M * 2 * p.Fp * (d->dtype == RDFC_F32 ? 4 : 2) + 255) / 256 * 256;
    p.bias_floats = ((size_t)p.row_blocks * 2 * p.Fp + 63) / 64 * 64;
    p.w_floats = ((size_t)p.splits * 2 * p.Fp * d->K + 63) / 64 * 64;
    p.dx_floats = p.dx_splits > 1 ? (size_t)p.dx_splits * d->M * d->K : 0;
    return p;
}
int check(const rdfc_gated_desc *d, const char *name) {
    RDFC_REQUIRE(d != nullptr, "%s: null descriptor", name);
    RDFC_REQUIRE(rdfc_dtype_ok(d->dtype), "%s: unsupported dtype %d", name, d->dtype);
    RDFC_REQUIRE(d->M >= 0 && d->M <= (int64_t)0x7fffffff * 32 && d->K > 0 && d->F > 0 && d->F <= (1 << 20) && d->K <= (1 << 20),
                 "%s: bad sizes M=%lld K=%d F=%d", name, (long long)d->M, d->K, d->F);
    RDFC_REQUIRE((int64_t)d->F * d->K <= (1ll << 36), "%s: weights of %d x %d are too large", name, d->F, d->K);
    RDFC_REQUIRE(d->ldx >= d->K && d->ldwg >= d->K && d->ldwu >= d->K, "%s: ld smaller than K", name);
    RDFC_REQUIRE(d->act == RDFC_ACT_RELU || d->act == RDFC_ACT_SIGMOID || d->act == RDFC_GATE_SILU || d->act == RDFC_GATE_GELU, "%s: unsupported activation %d",
                 name, d->act);
    return 0;
}
GLArgs args(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, const float *bg, const float *bu) {
    GLArgs p = {};
    p.x = x;
    p.wg = wg;
    p.wu = wu;
    p.bg = bg;
    p.bu = bu;
    p.M = d->M;
    p.K = d->K;
    p.Kv = (d->K + rdfc_vec(d->dtype) - 1) / rdfc_vec(d->dtype) * rdfc_vec(d->dtype);
    p.F = d->F;
    p.Fp = (d->F + 31) / 32 * 32;
    p.ldx = d->ldx;
    p.ldwg = d->ldwg;
    p.ldwu = d->ldwu;
    p.act = d->act;
    return p;
}

}  // namespace

extern "C" int rdfc_gated_linear(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, const float *bg, const float *bu, void *scratch,
                                 void *z, float *pre, void *stream) {
    if (check(d, "rdfc_gated_linear")) return 1;
    if (d->M == 0) return 0;
    RDFC_REQUIRE(x && wg && wu && z, "rdfc_gated_linear: null pointer");
    RDFC_REQUIRE(!bg == !bu, "rdfc_gated_linear: one bias without the other");
    const Packs k = packs_of(d, x, wg, wu);
    RDFC_REQUIRE(k.bytes() == 0 || (scratch && (reinterpret_cast<size_t>(scratch) & 15) == 0), "rdfc_gated_linear: these operands need (aligned) scratch memory");
    GLArgs p = args(d, x, wg, wu, bg, bu);
    if (pack(d, k, p, scratch, (hipStream_t)stream, "rdfc_gated_linear (pack)")) return 2;
    RDFC_REQUIRE(!pre || (d->dtype == RDFC_F32 && (reinterpret_cast<size_t>(pre) & 15) == 0), "rdfc_gated_linear: pre is kept for f32 maps, 16-byte aligned");
    p.z = z;
    p.pre = pre;
    const Tile t = tile_of([&](Tile t) { return cdiv(d->F, t.wtp) * (int64_t)cdiv(d->M, 2 * t.wtq); }, d->K >= 768);
    return launch_dma<FWD>(p, d->dtype, t, cdiv(d->F, t.wtp), cdiv(d->M, 2 * t.wtq), (hipStream_t)stream, "rdfc_gated_linear");
}

extern "C" size_t rdfc_gated_linear_scratch_bytes(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, int backward) {
    if (check(d, "rdfc_gated_linear_scratch_bytes")) return 0;
    const size_t k = packs_of(d, x, wg, wu).bytes();
    if (!backward) return k;
    const Plan q = plan_of(d);
    return k + q.d_bytes + 4 * (q.bias_floats + (q.w_floats > q.dx_floats ? q.w_floats : q.dx_floats));
}

extern "C" int rdfc_gated_linear_backward(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, const float *bg, const float *bu,
                                          const float *pre, const void *dz, int lddz, void *scratch, void *dx, void *dwg, void *dwu, int dw_dtype, float *dbg, float *dbu,
                                          void *stream) {
    if (check(d, "rdfc_gated_linear_backward")) return 1;
    RDFC_REQUIRE(lddz >= d->F, "rdfc_gated_linear_backward: lddz smaller than F");
    RDFC_REQUIRE(!bg == !bu, "rdfc_gated_linear_backward: one bias without the other");
    RDFC_REQUIRE(dw_dtype == RDFC_F32 || dw_dtype == d->dtype, "rdfc_gated_linear_backward: weight gradients are f32 or of the map's type");
    RDFC_REQUIRE(wg && wu && (d->M == 0 || (x && dz && scratch)), "rdfc_gated_linear_backward: null pointer");
    RDFC_REQUIRE(((reinterpret_cast<size_t>(scratch) | reinterpret_cast<size_t>(pre)) & 15) == 0, "rdfc_gated_linear_backward: scratch or pre is not 16-byte aligned");
    const Plan q = plan_of(d);
    const Packs k = packs_of(d, x, wg, wu);
    const hipStream_t st = (hipStream_t)stream;
    GLArgs p = args(d, x, wg, wu, bg, bu);
    p.dz = dz;
    p.lddz = lddz;
    p.D = (unsigned char *)scratch + k.bytes();
    float *bias = reinterpret_cast<float *>((unsigned char *)p.D + q.d_bytes), *w = bias + q.bias_floats;
    int row_blocks = 0;
    if (d->M > 0) {
        if (pack(d, k, p, scratch, st, "rdfc_gated_linear_backward (pack)")) return 2;
        p.partial = dbg || dbu ? bias : nullptr;
        if (d->dtype == RDFC_F32) {
            RDFC_REQUIRE(pre, "rdfc_gated_linear_backward: f32 maps need the forward pass's pre");
            p.pre = const_cast<float *>(pre);
            row_blocks = cdiv(d->M, ACT_ROWS);
            gated_act_kernel<<<dim3(row_blocks, cdiv(q.Fp, 256)), NT, 0, st>>>(p);
            RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (activation)");
        } else {
            row_blocks = cdiv(d->M, 2 * q.gated.wtq);
            if (launch_dma<BWD>(p, d->dtype, q.gated, cdiv(q.Fp, q.gated.wtp), row_blocks, st, "rdfc_gated_linear_backward")) return 2;
        }
        if (dx) {
            p.dx = dx;
            p.partial = q.dx_splits > 1 ? w : nullptr;           // (the weight gradients' parts follow in the same memory)
            p.split_rows = q.dx_cols;
            if (launch_dma<DX>(p, d->dtype, q.dx, cdiv(d->K, 2 * q.dx.wtp) * q.dx_splits, cdiv(d->M, 2 * q.dx.wtq), st, "rdfc_gated_linear_backward (input)")) return 2;
            if (q.dx_splits > 1) {
                const size_t n = (size_t)d->M * d->K;
                RDFC_DISPATCH(d->dtype, (join<T>(w, q.dx_splits, n, n, (T *)dx, nullptr, 1, st)));
                RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (input join)");
            }
        }
        if (dwg || dwu) {
            p.partial = w;
            p.split_rows = q.split_rows;
            const int tiles = cdiv(d->K, 2 * q.dw.wtp) * cdiv(2 * q.Fp, 2 * q.dw.wtq);
            if (launch_dma<DW>(p, d->dtype, q.dw, tiles, q.splits, st, "rdfc_gated_linear_backward (weights)")) return 2;
        }
    }
    // (M = 0: no parts, zeros)
    if (dbg || dbu) {
        gated_bias_kernel<<<2 * q.Fp / 32, 512, 0, st>>>(bias, row_blocks, d->F, q.Fp, dbg, dbu);
        RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (bias join)");
    }
    if (dwg || dwu) {
        RDFC_DISPATCH(dw_dtype, (join<T>(w, d->M > 0 ? q.splits : 0, (size_t)d->F * d->K, (size_t)2 * q.Fp * d->K, (T *)dwg, (T *)dwu, 2, st)));
        RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (join)");
    }
    return 0;
}
