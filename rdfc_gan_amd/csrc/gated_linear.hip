// gated_linear.hip -- the gated projection of a feed-forward block on pixel-major maps, and its backward pass:
//
//     g = x Wg^T + bg,  u = x Wu^T + bu,  z = act(g) * u            x [M][K], Wg, Wu [F][K], z [M][F]
//
// Forward: one product whose weight rows alternate 16 of Wg with 16 of Wu, so that a lane's accumulators hold g and u of the same
// elements and the activation and the product happen in registers: g and u never reach memory.
// Backward: the same product again, with dz in the epilogue: dg = dz u act'(g) and du = dz act(g), side by side in one map
// D [M][2 Fp] (Fp = F rounded up to 8, the columns between zero), with the bias gradients' partial sums in f32 beside the rounding to
// the map's type.  Then dx = D [Wg; Wu] and [dWg; dWu] = D^T x, the latter split over the pixels and joined in a fixed order.
#include "common.h"

namespace {

constexpr int NT = 256, BM = 64, BK = 32;

enum { FWD, BWD, DX, DW };

struct GLArgs {
    const void *x, *wg, *wu, *dz;
    const float *bg, *bu;
    void *z, *D, *dx;
    float *partial;                  // BWD: bias sums [row block][2 Fp];  DW: [split][2 Fp][K]
    int64_t M;
    int K, F, Fp, ldx, ldwg, ldwu, lddz, act;
    int64_t split_rows;              // DW: pixels per split
};

// ---- activation of the gate and its derivative (expf / erff: 1-2 ulp) --------------------------------------------------------
template <int ACT> __device__ __forceinline__ void gate_act(float g, float &a, float &da) {
    if constexpr (ACT == RDFC_ACT_RELU) {
        a = g > 0.f ? g : (g != g ? g : 0.f);
        da = g > 0.f ? 1.f : 0.f;
    } else if constexpr (ACT == RDFC_GATE_GELU) {
        const float phi = 0.5f * (1.f + erff(g * 0.70710678118654752f));
        a = g * phi;
        da = fmaf(g * 0.39894228040143268f, expf(-0.5f * g * g), phi);
    } else {
        const float s = 1.f / (1.f + expf(-g));
        a = ACT == RDFC_ACT_SIGMOID ? s : g * s;
        da = ACT == RDFC_ACT_SIGMOID ? s * (1.f - s) : s * fmaf(g, 1.f - s, 1.f);
    }
}
__device__ __forceinline__ void gate_act(int act, float g, float &a, float &da) {
    if (act == RDFC_ACT_RELU) gate_act<RDFC_ACT_RELU>(g, a, da);
    else if (act == RDFC_GATE_GELU) gate_act<RDFC_GATE_GELU>(g, a, da);
    else if (act == RDFC_ACT_SIGMOID) gate_act<RDFC_ACT_SIGMOID>(g, a, da);
    else gate_act<RDFC_GATE_SILU>(g, a, da);
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

// 64 x 64 tile, four waves of 32 x 32; operands element by element into LDS, any stride and alignment.
// P: rows of the MFMA (the output's contiguous dimension), Q: its columns.
template <typename T, int MODE> __global__ __launch_bounds__(NT) void gated_tile_kernel(GLArgs p) {
    constexpr int LDK = BK + 8;
    __shared__ T Ps[BM][LDK], Qs[BM][LDK];
    __shared__ float bsum[2][2][BM];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wp = wave >> 1, wq = wave & 1;
    const int64_t q0 = (int64_t)blockIdx.x * BM;
    const int p0 = blockIdx.y * (MODE == FWD || MODE == BWD ? BM / 2 : BM);
    const int64_t kbeg = MODE == DW ? blockIdx.z * p.split_rows : 0;
    const int64_t kend = MODE == DW ? min(kbeg + p.split_rows, p.M) : (MODE == DX ? 2 * p.Fp : p.K);
    const T *x = (const T *)p.x, *wg = (const T *)p.wg, *wu = (const T *)p.wu, *D = (const T *)p.D;
    auto fetch_p = [&](int r, int64_t k) -> T {
        if (k >= kend) return (T)0.f;
        if constexpr (MODE == FWD || MODE == BWD) {
            const int f = p0 + (r >> 5) * 16 + (r & 15);
            if (f >= p.F) return (T)0.f;
            return (r >> 4) & 1 ? wu[(size_t)f * p.ldwu + k] : wg[(size_t)f * p.ldwg + k];
        } else if constexpr (MODE == DX) {
            const int kk = p0 + r, f = (int)(k < p.Fp ? k : k - p.Fp);
            if (kk >= p.K || f >= p.F) return (T)0.f;
            return k < p.Fp ? wg[(size_t)f * p.ldwg + kk] : wu[(size_t)f * p.ldwu + kk];
        } else {
            return p0 + r < p.K ? x[k * p.ldx + p0 + r] : (T)0.f;
        }
    };
    auto fetch_q = [&](int r, int64_t k) -> T {
        if (k >= kend) return (T)0.f;
        if constexpr (MODE == FWD || MODE == BWD) return q0 + r < p.M ? x[(q0 + r) * p.ldx + k] : (T)0.f;
        else if constexpr (MODE == DX) return q0 + r < p.M ? D[(q0 + r) * 2 * p.Fp + k] : (T)0.f;
        else return q0 + r < 2 * p.Fp ? D[k * 2 * p.Fp + q0 + r] : (T)0.f;
    };
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    for (int64_t k0 = kbeg; k0 < kend; k0 += BK) {
        __syncthreads();
        for (int e = 0; e < 8; ++e) {
            // (neighbouring threads take neighbouring addresses: along k for the row layouts, along r for the others)
            int r, k;
            if (MODE == DW) r = tid & 63, k = (tid >> 6) + 4 * e;
            else r = (tid >> 5) + 8 * e, k = tid & 31;
            Qs[r][k] = fetch_q(r, k0 + k);
            if (MODE == DX) r = tid & 63, k = (tid >> 6) + 4 * e;
            Ps[r][k] = fetch_p(r, k0 + k);
        }
        __syncthreads();
        if constexpr (sizeof(T) == 2) {
            bf16x8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *reinterpret_cast<const bf16x8 *>(&Ps[wp * 32 + 16 * i + (lane & 15)][(lane >> 4) * 8]);
                b[i] = *reinterpret_cast<const bf16x8 *>(&Qs[wq * 32 + 16 * i + (lane & 15)][(lane >> 4) * 8]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma16<DtOf<T>::value>(a[i], b[j], acc[i][j]);
        } else {
            for (int k = 0; k < BK; k += 4) {
                float a[2], b[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    a[i] = Ps[wp * 32 + 16 * i + (lane & 15)][k + (lane >> 4)];
                    b[i] = Qs[wq * 32 + 16 * i + (lane & 15)][k + (lane >> 4)];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[j], acc[i][j], 0, 0, 0);
            }
        }
    }
    const int q4 = (lane >> 4) * 4;
    if constexpr (MODE == FWD || MODE == BWD) {
        const int f0 = p0 + wp * 16 + q4;
        float sg[4] = {0.f, 0.f, 0.f, 0.f}, su[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t m = q0 + wq * 32 + 16 * j + (lane & 15);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = f0 + r;
                if (m >= p.M || f >= p.Fp) continue;
                const bool in = f < p.F;
                const float g = acc[0][j][r] + (p.bg && in ? p.bg[f] : 0.f), u = acc[1][j][r] + (p.bu && in ? p.bu[f] : 0.f);
                float a, da;
                gate_act(p.act, g, a, da);
                if constexpr (MODE == FWD) {
                    if (in) Elem<T>::st((T *)p.z + m * p.F + f, a * u);
                } else {
                    const float dz = in ? Elem<T>::ld((const T *)p.dz + m * p.lddz + f) : 0.f;
                    const float dg = in ? dz * u * da : 0.f, du = in ? dz * a : 0.f;
                    Elem<T>::st((T *)p.D + m * 2 * p.Fp + f, dg);
                    Elem<T>::st((T *)p.D + m * 2 * p.Fp + p.Fp + f, du);
                    sg[r] += dg;
                    su[r] += du;
                }
            }
        }
        if constexpr (MODE == BWD) {
            if (p.partial == nullptr) return;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float a = row16_sum(sg[r]), b = row16_sum(su[r]);
                if ((lane & 15) == 0) bsum[wq][0][wp * 16 + q4 + r] = a, bsum[wq][1][wp * 16 + q4 + r] = b;
            }
            __syncthreads();
            if (tid < BM) {
                const int f = p0 + (tid & 31), kind = tid >> 5;
                if (f < p.Fp) p.partial[(size_t)blockIdx.x * 2 * p.Fp + kind * p.Fp + f] = bsum[0][kind][tid & 31] + bsum[1][kind][tid & 31];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t q = q0 + wq * 32 + 16 * j + (lane & 15);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int kk = p0 + wp * 32 + 16 * i + q4 + r;
                    if (kk >= p.K) continue;
                    if (MODE == DX && q < p.M) Elem<T>::st((T *)p.dx + q * p.K + kk, acc[i][j][r]);
                    if (MODE == DW && q < 2 * p.Fp) p.partial[((size_t)blockIdx.z * 2 * p.Fp + q) * p.K + kk] = acc[i][j][r];
                }
            }
    }
}

// out[kind][f][k] = sum over parts of partial[part][kind * Fp + f][k], in the order of the parts
template <typename TO> __global__ __launch_bounds__(NT) void gated_join_kernel(const float *__restrict__ partial, int parts, int F, int Fp, int K, TO *o0, TO *o1) {
    const size_t n = (size_t)F * K, i = (size_t)blockIdx.x * NT + threadIdx.x;
    if (i >= n) return;
    const size_t step = (size_t)2 * Fp * K, src = (size_t)blockIdx.y * Fp * K + i;
    TO *o = blockIdx.y ? o1 : o0;
    if (o == nullptr) return;
    double s = 0.;
    for (int k = 0; k < parts; ++k) s += (double)partial[k * step + src];
    Elem<TO>::st(o + i, (float)s);
}

struct Plan {
    int Fp, row_blocks, splits;
    int64_t split_rows;
    size_t d_bytes, bias_floats, w_floats;
};
Plan plan_of(const rdfc_gated_desc *d) {
    Plan p;
    p.Fp = (d->F + 7) / 8 * 8;
    p.row_blocks = (int)((d->M + BM - 1) / BM);
    const int64_t tiles = (int64_t)cdiv(2 * p.Fp, BM) * cdiv(d->K, BM);
    int64_t s = 1024 / tiles;
    const int64_t most = (d->M + 511) / 512;
    s = s < 1 ? 1 : s > most ? most : s;
    s = s < 1 ? 1 : s;
    p.split_rows = ((d->M + s - 1) / s + BK - 1) / BK * BK;
    if (p.split_rows < BK) p.split_rows = BK;
    p.splits = (int)((d->M + p.split_rows - 1) / p.split_rows);
    p.d_bytes = ((size_t)d->M * 2 * p.Fp * (d->dtype == RDFC_F32 ? 4 : 2) + 255) / 256 * 256;
    p.bias_floats = ((size_t)p.row_blocks * 2 * p.Fp + 63) / 64 * 64;
    p.w_floats = (size_t)p.splits * 2 * p.Fp * d->K;
    return p;
}
int check(const rdfc_gated_desc *d, const char *name) {
    RDFC_REQUIRE(d != nullptr, "%s: null descriptor", name);
    RDFC_REQUIRE(rdfc_dtype_ok(d->dtype), "%s: unsupported dtype %d", name, d->dtype);
    RDFC_REQUIRE(d->M >= 0 && d->M <= (int64_t)0x7fffffff * 32 && d->K > 0 && d->F > 0 && d->F <= (1 << 20) && d->K <= (1 << 20),
                 "%s: bad sizes M=%lld K=%d F=%d", name, (long long)d->M, d->K, d->F);
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
    p.F = d->F;
    p.Fp = (d->F + 7) / 8 * 8;
    p.ldx = d->ldx;
    p.ldwg = d->ldwg;
    p.ldwu = d->ldwu;
    p.act = d->act;
    return p;
}

}  // namespace

extern "C" int rdfc_gated_linear(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, const float *bg, const float *bu, void *z,
                                 void *stream) {
    if (check(d, "rdfc_gated_linear")) return 1;
    if (d->M == 0) return 0;
    RDFC_REQUIRE(x && wg && wu && z, "rdfc_gated_linear: null pointer");
    RDFC_REQUIRE(!bg == !bu, "rdfc_gated_linear: one bias without the other");
    GLArgs p = args(d, x, wg, wu, bg, bu);
    p.z = z;
    const dim3 grid(cdiv(d->M, BM), cdiv(d->F, BM / 2));
    RDFC_DISPATCH(d->dtype, (gated_tile_kernel<T, FWD><<<grid, NT, 0, (hipStream_t)stream>>>(p)));
    RDFC_LAUNCH_CHECK("rdfc_gated_linear");
    return 0;
}

extern "C" size_t rdfc_gated_linear_scratch_bytes(const rdfc_gated_desc *d) {
    if (check(d, "rdfc_gated_linear_scratch_bytes")) return 0;
    const Plan q = plan_of(d);
    return q.d_bytes + 4 * (q.bias_floats + q.w_floats);
}

extern "C" int rdfc_gated_linear_backward(const rdfc_gated_desc *d, const void *x, const void *wg, const void *wu, const float *bg, const float *bu,
                                          const void *dz, int lddz, void *scratch, void *dx, void *dwg, void *dwu, int dw_dtype, float *dbg, float *dbu,
                                          void *stream) {
    if (check(d, "rdfc_gated_linear_backward")) return 1;
    RDFC_REQUIRE(lddz >= d->F, "rdfc_gated_linear_backward: lddz smaller than F");
    RDFC_REQUIRE(!bg == !bu, "rdfc_gated_linear_backward: one bias without the other");
    RDFC_REQUIRE(dw_dtype == RDFC_F32 || dw_dtype == d->dtype, "rdfc_gated_linear_backward: weight gradients are f32 or of the map's type");
    RDFC_REQUIRE(wg && wu && (d->M == 0 || (x && dz && scratch)), "rdfc_gated_linear_backward: null pointer");
    const Plan q = plan_of(d);
    const hipStream_t st = (hipStream_t)stream;
    GLArgs p = args(d, x, wg, wu, bg, bu);
    p.dz = dz;
    p.lddz = lddz;
    p.D = scratch;
    float *bias = reinterpret_cast<float *>((unsigned char *)scratch + q.d_bytes), *w = bias + q.bias_floats;
    if (d->M > 0) {
        p.partial = dbg || dbu ? bias : nullptr;
        RDFC_DISPATCH(d->dtype, (gated_tile_kernel<T, BWD><<<dim3(q.row_blocks, cdiv(q.Fp, BM / 2)), NT, 0, st>>>(p)));
        RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward");
        if (dx) {
            p.dx = dx;
            RDFC_DISPATCH(d->dtype, (gated_tile_kernel<T, DX><<<dim3(q.row_blocks, cdiv(d->K, BM)), NT, 0, st>>>(p)));
            RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (input)");
        }
        if (dwg || dwu) {
            p.partial = w;
            p.split_rows = q.split_rows;
            RDFC_DISPATCH(d->dtype, (gated_tile_kernel<T, DW><<<dim3(cdiv(2 * q.Fp, BM), cdiv(d->K, BM), q.splits), NT, 0, st>>>(p)));
            RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (weights)");
        }
    }
    // (M = 0: no parts, zeros)
    if (dbg || dbu) {
        gated_join_kernel<float><<<dim3(cdiv(d->F, NT), 2), NT, 0, st>>>(bias, d->M > 0 ? q.row_blocks : 0, d->F, q.Fp, 1, dbg, dbu);
        RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (bias join)");
    }
    if (dwg || dwu) {
        const dim3 grid((unsigned)(((size_t)d->F * d->K + NT - 1) / NT), 2);
        RDFC_DISPATCH(dw_dtype, (gated_join_kernel<T><<<grid, NT, 0, st>>>(w, d->M > 0 ? q.splits : 0, d->F, q.Fp, d->K, (T *)dwg, (T *)dwu)));
        RDFC_LAUNCH_CHECK("rdfc_gated_linear_backward (join)");
    }
    return 0;
}
