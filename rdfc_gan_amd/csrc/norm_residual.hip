// norm_residual.hip -- the junction of a residual stream with a block's output, between two row norms:
//
//     u = N_post(h)                                      (or h)
//     y = x + scale[c] * gate[n][c] * dropout(u)         the residual stream behind the block
//     n = N_pre(y)                                       the next block's input
//
// N: RMS norm v * rsqrt(mean(v^2) + eps) * w or layer norm (v - mean(v)) * rsqrt(var(v) + eps) * w + b over the C channels of a pixel.
// A pixel's channels stay in the registers of the LPR lanes that own it from the load to the last store, so a pass moves x, h, y and n
// once (forward) or x, h, dy, dn, dx and dh once (backward): HBM is the bound.  The backward pass recomputes y from x and h (the
// same bytes as reading a saved y) in f32, so neither y nor the dropout mask nor the normalised maps are kept -- four f32 statistics
// per pixel are.
//
// Measured: 8x57x76x1024 f16 (layer norm before the next block) 51 us forward, 284 MB at 5.5 TB/s, and 102 backward, 426 MB at 4.2 TB/s (two waves a
// SIMD: 180 registers, the sums alone are 32; a second row fetched ahead changes nothing), column sums 10.  8x57x76x256 bf16, both norms, gate
// and dropout: 18 us forward, 25 backward and 8 for the column sums.
//
// Column sums (gradients of the four norm parameters, of scale and of gate) reduce to four sums per sample and channel:
//     A = sum D t hhat,  B = sum D t   (t: cotangent of y, D: dropout factor, hhat: normalised h, or h itself without N_post)
//     P = sum dn yhat,   Q = sum dn
// S = w A + b B is then the common part of d gate = scale S and d scale = sum_n gate S.  Each lane adds its own channels over
// its rows in f32, workgroups write one partial row each, and a second kernel adds those in a fixed order in f64: no atomics, the same
// bits every run.
#include "philox.h"

#include <initializer_list>

namespace {

// threads of a workgroup: four waves, or the two that share a row of up to 1024 channels (two vectors a lane of one wave would need 300 registers in
// the backward kernel)
constexpr int threads_of(int lpr) { return lpr == 128 ? 128 : 256; }

struct NRArgs {
    const void *x, *h;
    void *y, *n;
    const void *dy, *dn;
    void *dx, *dh;
    int64_t rows;                    // per sample
    int C, ldx, ldh, ldy, ldn, lddy, lddn;
    const float *gate, *scale, *post_w, *post_b, *pre_w, *pre_b;
    int layer, post, pre, par_al;    // par_al: every parameter vector is 16-byte aligned
    float eps;
    DropArgs drop;
    f32x4 *stats;                    // per row: mean and reciprocal deviation of h, of y
    float *partial;
    int64_t chunk;                   // rows per workgroup
};

// ---- sums over the LPR lanes that own a row ------------------------------------------------------------------------------
// All of it in vector registers (DPP inside 16 lanes, permlane swaps above): a shuffle through LDS has several times the latency, and a
// row's pass waits for up to four sums in turn.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// v of a lane + v of the lane W away (lane ^ W)
template <int W> __device__ __forceinline__ float halves_sum(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    unsigned r0, r1;                                             // (taken apart first: a bit cast of the vector's element 1 reads element 0)
    if constexpr (W == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        r0 = r[0], r1 = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        r0 = r[0], r1 = r[1];
    }
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
template <int LPR> __device__ __forceinline__ float lanes_sum(float v) {
    v = dpp_add<0xB1>(v);                                        // quad_perm 1,0,3,2
    v = dpp_add<0x4E>(v);                                        // quad_perm 2,3,0,1
    v = dpp_add<0x141>(v);                                       // row_half_mirror: eight lanes
    if constexpr (LPR >= 16) v = dpp_add<0x140>(v);              // row_mirror
    if constexpr (LPR >= 32) v = halves_sum<16>(v);
    if constexpr (LPR >= 64) v = halves_sum<32>(v);
    return v;
}
// two sums at once.  LPR > 64: over the workgroup, through LDS (`buf`: two slots of 8 floats used in turn; every thread calls)
template <int LPR> __device__ __forceinline__ void row_sum2(float &a, float &b, float (*buf)[8], int &turn) {
    a = lanes_sum<LPR>(a);
    b = lanes_sum<LPR>(b);
    if constexpr (LPR > 64) {
        float *s = buf[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
            s[threadIdx.x >> 6] = a;
            s[4 + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();                                         // (the other slot is not written again before the next barrier)
        a = LPR == 128 ? s[0] + s[1] : (s[0] + s[1]) + (s[2] + s[3]);
        b = LPR == 128 ? s[4] + s[5] : (s[4] + s[5]) + (s[6] + s[7]);
    }
}

// ---- eight channels ------------------------------------------------------------------------------------------------------
// as they lie in memory, so that a row can be fetched while the one before it is worked on.  ALIGNED: C is a multiple of 8 and every
// row 16-byte aligned
template <typename T, bool ALIGNED> struct Raw8 {
    static constexpr int NV = sizeof(T) / 2;
    Vec16<T> v[NV];
    __device__ __forceinline__ void load(const T *row, int c, int C) {
        if constexpr (ALIGNED) {
            if (c < C) {
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i].load(row + c + i * Elem<T>::VEC);
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i].zero();
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i / Elem<T>::VEC].set(i % Elem<T>::VEC, c + i < C ? Elem<T>::ld(row + c + i) : 0.f);
        }
    }
    __device__ __forceinline__ float get(int i) const { return v[i / Elem<T>::VEC].get(i % Elem<T>::VEC); }
    __device__ __forceinline__ void get8(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = get(i);
    }
};
template <typename T, bool ALIGNED> __device__ __forceinline__ void store8(const float (&v)[8], T *row, int c, int C) {
    if constexpr (ALIGNED) {
        if (c >= C) return;
        if constexpr (sizeof(T) == 4) {
            Vec16<T> a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) a.set(i, v[i]), b.set(i, v[4 + i]);
            a.store(row + c);
            b.store(row + c + 4);
        } else {
            Vec16<T> a;
#pragma unroll
            for (int i = 0; i < 8; ++i) a.set(i, v[i]);
            a.store(row + c);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < C) Elem<T>::st(row + c + i, v[i]);
    }
}
// a parameter vector (f32); a null pointer stands for `none`.  0 beyond C: what the lanes behind the last channel hold must not enter a sum
template <bool ALIGNED> __device__ __forceinline__ void load_par(float (&v)[8], const float *p, int c, int C, float none, int par_al) {
    if (ALIGNED && par_al && p != nullptr && c < C) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p + c), b = *reinterpret_cast<const f32x4 *>(p + c + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i >= C ? 0.f : p != nullptr ? p[c + i] : none;
}
// y = x + D (fw hhat + fb): fw = scale gate w_post, fb = scale gate b_post
template <int LPR, int VPL, bool ALIGNED> __device__ __forceinline__ void load_factors(const NRArgs &p, int li, float (&fw)[VPL][8], float (&fb)[VPL][8]) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int c = (v * LPR + li) * 8;
        float s[8], g[8];
        load_par<ALIGNED>(s, p.scale, c, p.C, 1.f, p.par_al);
        load_par<ALIGNED>(g, p.gate ? p.gate + (size_t)blockIdx.y * p.C : nullptr, c, p.C, 1.f, p.par_al);
        load_par<ALIGNED>(fw[v], p.post_w, c, p.C, 1.f, p.par_al);
        load_par<ALIGNED>(fb[v], p.post_b, c, p.C, 0.f, p.par_al);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            fw[v][i] *= s[i] * g[i];
            fb[v][i] *= s[i] * g[i];
        }
    }
}

template <typename T, int LPR, int VPL, bool ALIGNED>
__global__ __launch_bounds__(threads_of(LPR), VPL == 1 ? (sizeof(T) == 2 ? 5 : 4) : 1) void norm_residual_kernel(NRArgs p) {
    constexpr int NT = threads_of(LPR), RPB = NT / LPR;
    __shared__ float buf[2][8];
    int turn = 0;
    const int li = threadIdx.x % LPR, C = p.C;
    const float rC = 1.f / (float)C;
    const unsigned long long seed = p.drop.key ? p.drop.key[0] : p.drop.seed, offset = p.drop.key ? p.drop.key[1] : p.drop.offset;
    float fw[VPL][8], fb[VPL][8], qw[VPL][8], qb[VPL][8];
    load_factors<LPR, VPL, ALIGNED>(p, li, fw, fb);
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        load_par<ALIGNED>(qw[v], p.pre_w, (v * LPR + li) * 8, C, 1.f, p.par_al);
        load_par<ALIGNED>(qb[v], p.pre_b, (v * LPR + li) * 8, C, 0.f, p.par_al);
    }
    const int64_t r0 = (int64_t)blockIdx.x * p.chunk, r1 = min(r0 + p.chunk, p.rows), base = (int64_t)blockIdx.y * p.rows;
    // mean and reciprocal deviation of the row in a[][]; a[][] becomes the normalised row
    auto normalise = [&](float (&a)[VPL][8], float &mean, float &rstd) {
        mean = 0.f;
        float s = 0.f, z = 0.f;
        if (p.layer) {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) s += a[v][i];
            row_sum2<LPR>(s, z, buf, turn);
            mean = s * rC;
        }
        s = z = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[v][i] = (v * LPR + li) * 8 + i < C ? a[v][i] - mean : 0.f;
                s = fmaf(a[v][i], a[v][i], s);
            }
        row_sum2<LPR>(s, z, buf, turn);
        rstd = 1.f / sqrtf(s * rC + p.eps);
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) a[v][i] *= rstd;
    };
    Raw8<T, ALIGNED> nx[VPL], nh[VPL];                            // the next row
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            nx[v].load((const T *)p.x + (base + r) * p.ldx, (v * LPR + li) * 8, C);
            if (p.h != nullptr) nh[v].load((const T *)p.h + (base + r) * p.ldh, (v * LPR + li) * 8, C);
        }
    };
    // the row's mask, drawn before its data is touched: the multiplications run while the loads are under way
    auto draw = [&](int64_t row, unsigned (&keep)[VPL]) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            keep[v] = 0xff;
            if (p.drop.threshold != 0) {
                keep[v] = keep8<ALIGNED>((unsigned long long)row * C + (v * LPR + li) * 8, p.drop.threshold, seed, offset);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    int64_t r = r0 + threadIdx.x / LPR;
    if (r < r1) fetch(r);
    for (; r < r1; r += RPB) {
        const int64_t row = base + r;
        float a[VPL][8], b[VPL][8];
        unsigned keep[VPL];
        draw(row, keep);
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            nx[v].get8(a[v]);
            if (p.h != nullptr) nh[v].get8(b[v]);
        }
        if (r + RPB < r1) fetch(r + RPB);
        f32x4 st = {0.f, 0.f, 0.f, 0.f};
        if (p.h != nullptr) {
            if (p.post) {
                float m, s;
                normalise(b, m, s);
                st[0] = m;
                st[1] = s;
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int c = (v * LPR + li) * 8;
                // (a dropped element stays out whatever its value: no 0 * inf)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (keep[v] >> i & 1) a[v][i] = fmaf(fmaf(b[v][i], fw[v][i], fb[v][i]), p.drop.inv, a[v][i]);
                store8<T, ALIGNED>(a[v], (T *)p.y + row * p.ldy, c, C);
            }
        }
        if (p.pre) {
            float m, s;
            normalise(a, m, s);
            st[2] = m;
            st[3] = s;
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) a[v][i] = fmaf(a[v][i], qw[v][i], qb[v][i]);
                store8<T, ALIGNED>(a[v], (T *)p.n + row * p.ldn, (v * LPR + li) * 8, C);
            }
        }
        if (p.stats != nullptr && li == 0) p.stats[row] = st;
    }
}

template <typename T, int LPR, int VPL, bool ALIGNED>
__global__ __launch_bounds__(threads_of(LPR), VPL == 1 ? 2 : 1) void norm_residual_bwd_kernel(NRArgs p) {
    constexpr int NT = threads_of(LPR), RPB = NT / LPR;
    __shared__ float buf[2][8];
    __shared__ float red[LPR <= 64 ? 4 : 1][LPR <= 64 ? LPR * VPL * 8 : 1];
    int turn = 0;
    const int li = threadIdx.x % LPR, grp = threadIdx.x / LPR, C = p.C;
    const float rC = 1.f / (float)C;
    const unsigned long long seed = p.drop.key ? p.drop.key[0] : p.drop.seed, offset = p.drop.key ? p.drop.key[1] : p.drop.offset;
    float fw[VPL][8], fb[VPL][8], qw[VPL][8];
    float sum[4][VPL][8];                                        // A, B, P, Q
    load_factors<LPR, VPL, ALIGNED>(p, li, fw, fb);
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        load_par<ALIGNED>(qw[v], p.pre_w, (v * LPR + li) * 8, C, 1.f, p.par_al);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[k][v][i] = 0.f;
    }
    const int64_t r0 = (int64_t)blockIdx.x * p.chunk, r1 = min(r0 + p.chunk, p.rows), base = (int64_t)blockIdx.y * p.rows;
    // gradient through a row norm: g = cotangent of the normalised row (0 beyond C), hat = the normalised row
    auto through = [&](float (&g)[VPL][8], const float (&hat)[VPL][8], float rstd) {
        float s = 0.f, z = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s = fmaf(g[v][i], hat[v][i], s);
                z += g[v][i];
            }
        row_sum2<LPR>(s, z, buf, turn);
        s *= rC;
        z = p.layer ? z * rC : 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) g[v][i] = rstd * (g[v][i] - fmaf(hat[v][i], s, z));
    };
    Raw8<T, ALIGNED> nx[VPL], nh[VPL], ny[VPL], nn[VPL];          // the next row
    f32x4 nst = {0.f, 0.f, 0.f, 0.f};
    auto fetch = [&](int64_t r) {
        nst = p.stats[base + r];
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c = (v * LPR + li) * 8;
            nx[v].load((const T *)p.x + (base + r) * p.ldx, c, C);
            if (p.h != nullptr) nh[v].load((const T *)p.h + (base + r) * p.ldh, c, C);
            if (p.dy != nullptr) ny[v].load((const T *)p.dy + (base + r) * p.lddy, c, C);
            if (p.dn != nullptr) nn[v].load((const T *)p.dn + (base + r) * p.lddn, c, C);
        }
    };
    // the row's mask, drawn before its data is touched: the multiplications run while the loads are under way
    auto draw = [&](int64_t row, unsigned (&keep)[VPL]) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            keep[v] = 0xff;
            if (p.drop.threshold != 0) {
                keep[v] = keep8<ALIGNED>((unsigned long long)row * C + (v * LPR + li) * 8, p.drop.threshold, seed, offset);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    int64_t r = r0 + grp;
    if (r < r1) fetch(r);
    for (; r < r1; r += RPB) {
        const int64_t row = base + r;
        float a[VPL][8], hat[VPL][8], t[VPL][8];
        Raw8<T, ALIGNED> dy[VPL];
        unsigned keep[VPL];
        draw(row, keep);
        const f32x4 st = nst;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            nx[v].get8(a[v]);
            if (p.h != nullptr) nh[v].get8(hat[v]);
            if (p.dn != nullptr) nn[v].get8(t[v]);
            if (p.dy != nullptr) dy[v] = ny[v];
        }
        if (r + RPB < r1) fetch(r + RPB);
        // hat = normalised h (or h), a = y
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c = (v * LPR + li) * 8;
            if (p.h != nullptr) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (p.post) hat[v][i] = c + i < C ? (hat[v][i] - st[0]) * st[1] : 0.f;
                    if (keep[v] >> i & 1) a[v][i] = fmaf(fmaf(hat[v][i], fw[v][i], fb[v][i]), p.drop.inv, a[v][i]);
                }
            }
        }
        // t = cotangent of y
        if (p.dn != nullptr) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const int c = (v * LPR + li) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[v][i] = c + i < C ? (a[v][i] - st[2]) * st[3] : 0.f;
                    sum[2][v][i] = fmaf(t[v][i], a[v][i], sum[2][v][i]);
                    sum[3][v][i] += t[v][i];
                    t[v][i] *= qw[v][i];
                }
            }
            through(t, a, st[3]);
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) t[v][i] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const int c = (v * LPR + li) * 8;
            if (p.dy != nullptr) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[v][i] += dy[v].get(i);
            }
            store8<T, ALIGNED>(t[v], (T *)p.dx + row * C, c, C);
        }
        if (p.h == nullptr) continue;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool kept = keep[v] >> i & 1;
                const float d = kept ? t[v][i] * p.drop.inv : 0.f;
                sum[0][v][i] = kept ? fmaf(d, hat[v][i], sum[0][v][i]) : sum[0][v][i];      // (a dropped element may hold anything)
                sum[1][v][i] += d;
                t[v][i] = d * fw[v][i];
            }
        if (p.post) through(t, hat, st[1]);
#pragma unroll
        for (int v = 0; v < VPL; ++v) store8<T, ALIGNED>(t[v], (T *)p.dh + row * C, (v * LPR + li) * 8, C);
    }
    // the row groups' sums: those of a wave in its registers, the four waves' in LDS, one partial row per sum: partial[sample][chunk][4][C]
    if (p.partial == nullptr) return;
    float *out = p.partial + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 * C;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (LPR > 64) {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((v * LPR + li) * 8 + i < C) out[(size_t)k * C + (v * LPR + li) * 8 + i] = sum[k][v][i];
        } else {
            if (k) __syncthreads();
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float &s = sum[k][v][i];
                    if constexpr (LPR <= 8) s = dpp_add<0x128>(s);           // row_ror:8
                    if constexpr (LPR <= 16) s = halves_sum<16>(s);
                    if constexpr (LPR <= 32) s = halves_sum<32>(s);
                }
                if ((threadIdx.x & 63) < LPR) {
                    f32x4 *dst = reinterpret_cast<f32x4 *>(&red[threadIdx.x >> 6][(v * LPR + li) * 8]);
                    dst[0] = f32x4{sum[k][v][0], sum[k][v][1], sum[k][v][2], sum[k][v][3]};
                    dst[1] = f32x4{sum[k][v][4], sum[k][v][5], sum[k][v][6], sum[k][v][7]};
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += NT) out[(size_t)k * C + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
        }
    }
}

// ---- column sums ---------------------------------------------------------------------------------------------------------
// Two small kernels.  First, 64 columns x 8 row lanes per workgroup over PARTS slices of a sample's partial rows (one workgroup per
// column tile alone reads 256 B of every row: at 20 GB/s a CU a thousand rows took 30 us); then one thread per channel.
struct NRGrads {
    float *gate, *scale, *post_w, *post_b, *pre_w, *pre_b;       // each may be null
};
constexpr int SUM_COLS = 64, SUM_ROWS = 8, SLICE = 128;          // partial rows per workgroup
__global__ __launch_bounds__(SUM_COLS * SUM_ROWS) void norm_residual_sum_kernel(const float *__restrict__ partial, double *__restrict__ sums, int cols, int nchunk) {
    __shared__ double red[SUM_ROWS][SUM_COLS];
    const int cl = threadIdx.x % SUM_COLS, rl = threadIdx.x / SUM_COLS, c = blockIdx.x * SUM_COLS + cl;
    const int k0 = blockIdx.z * SLICE, k1 = min(k0 + SLICE, nchunk);
    double s = 0.;
    if (c < cols) {
        const float *src = partial + (size_t)blockIdx.y * nchunk * cols + c;
#pragma unroll 8
        for (int k = k0 + rl; k < k1; k += SUM_ROWS) s += (double)src[(size_t)k * cols];
    }
    red[rl][cl] = s;
    __syncthreads();
    if (rl != 0 || c >= cols) return;
#pragma unroll
    for (int k = 1; k < SUM_ROWS; ++k) s += red[k][cl];
    sums[((size_t)blockIdx.y * gridDim.z + blockIdx.z) * cols + c] = s;
}
// 64 channels x 8 sample lanes
__global__ __launch_bounds__(512) void norm_residual_grads_kernel(NRArgs p, NRGrads o, const double *__restrict__ sums, int samples, int slices) {
    __shared__ double red[8][5][64];
    const int C = p.C, cl = threadIdx.x & 63, gl = threadIdx.x >> 6, c = blockIdx.x * 64 + cl;
    double acc[5] = {0., 0., 0., 0., 0.};                        // scale, post_w, post_b, pre_w, pre_b
    if (c < C) {
        const double sc = p.scale ? p.scale[c] : 1., w = p.post && p.post_w ? p.post_w[c] : 1., b = p.post && p.post_b ? p.post_b[c] : 0.;
        for (int g = gl; g < samples; g += 8) {
            double s[4] = {0., 0., 0., 0.};
#pragma unroll 4
            for (int k = 0; k < slices; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += sums[(((size_t)g * slices + k) * 4 + j) * C + c];
            const double gt = p.gate ? p.gate[(size_t)g * C + c] : 1., S = w * s[0] + b * s[1];
            if (o.gate) o.gate[(size_t)g * C + c] = (float)(sc * S);
            acc[0] += gt * S;
            acc[1] += sc * gt * s[0];
            acc[2] += sc * gt * s[1];
            acc[3] += s[2];
            acc[4] += s[3];
        }
    }
#pragma unroll
    for (int k = 0; k < 5; ++k) red[gl][k][cl] = acc[k];
    __syncthreads();
    if (gl >= 5 || c >= C) return;
    double s = 0.;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += red[k][gl][cl];
    float *out = gl == 0 ? o.scale : gl == 1 ? o.post_w : gl == 2 ? o.post_b : gl == 3 ? o.pre_w : o.pre_b;
    if (out) out[c] = (float)s;
}

constexpr int MAXC = 8192;
// lanes and vectors of eight channels per lane: the fewest lanes that hold a row
template <typename F> void with_layout(int C, F &&f) {
    const int nv = (C + 7) / 8;
    if (nv <= 8) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    else if (nv <= 16) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    else if (nv <= 32) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
    else if (nv <= 64) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (nv <= 128) f(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
    else if (nv <= 256) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (nv <= 512) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
}
int lanes_of(int C) {
    int l = 0;
    with_layout(C, [&](auto lpr, auto) { l = decltype(lpr)::value; });
    return l;
}
// rows per workgroup: about `groups` workgroups in all (the backward kernel leaves 4 C sums per workgroup)
int64_t chunk_of(int64_t rows, int samples, int C, int groups) {
    const int lpr = lanes_of(C), nt = threads_of(lpr);
    const int64_t rpb = nt / lpr, total = rows * samples;
    groups *= 256 / nt;
    int64_t per = (total + groups - 1) / groups;
    per = (per + rpb - 1) / rpb * rpb;
    while ((rows + per - 1) / per >= (1 << 20)) per *= 2;
    return per;
}
// (both: what the chip holds at once -- five and two waves a SIMD -- in one round.  The backward kernel at three waves spills, and a second round that is
// not full costs more than the waves give: x1024 f16 at 768 / 512 workgroups of three / two waves 127 / 111 us)
constexpr int FWD_GROUPS = 1280, BWD_GROUPS = 512;
struct NRChunks {
    int64_t chunk;
    int nchunk, slices;
    size_t partial, sums;            // floats of the partial rows (even), doubles of their sums
};
NRChunks bwd_chunks(int64_t rows, int samples, int C) {
    NRChunks k;
    k.chunk = chunk_of(rows, samples, C, BWD_GROUPS);
    k.nchunk = (int)((rows + k.chunk - 1) / k.chunk);
    k.slices = (k.nchunk + SLICE - 1) / SLICE;
    k.partial = (size_t)samples * k.nchunk * 4 * C;
    k.sums = (size_t)samples * k.slices * 4 * C;
    return k;
}
bool par_aligned(std::initializer_list<const float *> ps) {
    size_t a = 0;
    for (const float *p : ps) a |= reinterpret_cast<size_t>(p);
    return a % 16 == 0;
}
bool row_aligned(const void *p, int ld, int dtype) { return (reinterpret_cast<size_t>(p) & 15) == 0 && ld % rdfc_vec(dtype) == 0; }

}  // namespace

static int nr_check(const rdfc_norm_residual_desc *d, const char *name) {
    RDFC_REQUIRE(d != nullptr, "%s: null descriptor", name);
    RDFC_REQUIRE(rdfc_dtype_ok(d->dtype), "%s: unsupported dtype %d", name, d->dtype);
    RDFC_REQUIRE(d->samples >= 0 && d->samples <= 65535 && d->rows >= 0, "%s: bad sizes samples=%d rows=%lld", name, d->samples, (long long)d->rows);
    RDFC_REQUIRE(d->C > 0 && d->C <= MAXC, "%s: C = %d is not in [1, %d]", name, d->C, MAXC);
    RDFC_REQUIRE(d->ldx >= d->C && d->ldh >= d->C, "%s: ld smaller than C", name);
    RDFC_REQUIRE(d->threshold >= 0 && d->threshold <= 65536, "%s: threshold %d is not in [0, 65536]", name, d->threshold);
    return 0;
}
static NRArgs nr_args(const rdfc_norm_residual_desc *d, const void *x, const void *h, const float *gate, const float *scale, const float *post_w,
                      const float *post_b, const float *pre_w, const float *pre_b, const uint64_t *key) {
    NRArgs p = {};
    p.x = x;
    p.h = h;
    p.rows = d->rows;
    p.C = d->C;
    p.ldx = d->ldx;
    p.ldh = d->ldh;
    p.gate = gate;
    p.scale = scale;
    p.post_w = post_w;
    p.post_b = post_b;
    p.pre_w = pre_w;
    p.pre_b = pre_b;
    p.layer = d->layer;
    p.post = d->post && h != nullptr;
    p.pre = d->pre;
    p.eps = d->eps;
    p.par_al = par_aligned({gate, scale, post_w, post_b, pre_w, pre_b});
    drop_args(p.drop, d->threshold, d->seed, d->offset, key);
    return p;
}

extern "C" int rdfc_norm_residual(const rdfc_norm_residual_desc *d, const void *x, const void *h, const float *gate, const float *scale,
                                  const float *post_w, const float *post_b, const float *pre_w, const float *pre_b, const uint64_t *key, void *y,
                                  void *n, float *stats, void *stream) {
    if (nr_check(d, "rdfc_norm_residual")) return 1;
    if (d->samples == 0 || d->rows == 0) return 0;
    RDFC_REQUIRE((reinterpret_cast<size_t>(stats) & 15) == 0, "rdfc_norm_residual: stats is not 16-byte aligned");
    RDFC_REQUIRE(x && (h ? y != nullptr : (d->pre && !gate && !scale)) && (!d->pre || n), "rdfc_norm_residual: null map");
    NRArgs p = nr_args(d, x, h, gate, scale, post_w, post_b, pre_w, pre_b, key);
    p.y = y;
    p.n = n;
    p.ldy = p.ldn = d->C;
    p.stats = reinterpret_cast<f32x4 *>(stats);
    // (without a gate the samples are one run of rows)
    const int samples = gate ? d->samples : 1;
    p.rows = gate ? d->rows : d->rows * d->samples;
    p.chunk = chunk_of(p.rows, samples, d->C, FWD_GROUPS);
    const dim3 grid((unsigned)((p.rows + p.chunk - 1) / p.chunk), samples);
    const bool al = row_aligned(x, d->ldx, d->dtype) && row_aligned(h, d->ldh, d->dtype) && row_aligned(y, d->C, d->dtype) && row_aligned(n, d->C, d->dtype) && d->C % 8 == 0;
    with_layout(d->C, [&](auto lpr, auto vpl) {
        constexpr int L = decltype(lpr)::value, V = decltype(vpl)::value;
        RDFC_DISPATCH(d->dtype, if (al) norm_residual_kernel<T, L, V, true><<<grid, threads_of(L), 0, (hipStream_t)stream>>>(p);
                      else norm_residual_kernel<T, L, V, false><<<grid, threads_of(L), 0, (hipStream_t)stream>>>(p));
    });
    RDFC_LAUNCH_CHECK("rdfc_norm_residual");
    return 0;
}

extern "C" size_t rdfc_norm_residual_scratch_floats(const rdfc_norm_residual_desc *d, int gated) {
    if (nr_check(d, "rdfc_norm_residual_scratch_floats") || d->samples == 0 || d->rows == 0) return 0;
    const int samples = gated ? d->samples : 1;
    const NRChunks k = bwd_chunks(gated ? d->rows : d->rows * d->samples, samples, d->C);
    return k.partial + 2 * k.sums;
}

extern "C" int rdfc_norm_residual_backward(const rdfc_norm_residual_desc *d, const void *x, const void *h, const float *gate, const float *scale,
                                           const float *post_w, const float *post_b, const float *pre_w, const uint64_t *key, const float *stats,
                                           const void *dy, int lddy, const void *dn, int lddn, void *dx, void *dh, float *scratch, float *d_gate,
                                           float *d_scale, float *d_post_w, float *d_post_b, float *d_pre_w, float *d_pre_b, void *stream) {
    if (nr_check(d, "rdfc_norm_residual_backward")) return 1;
    RDFC_REQUIRE(!dy || lddy >= d->C, "rdfc_norm_residual_backward: lddy smaller than C");
    RDFC_REQUIRE(!dn || lddn >= d->C, "rdfc_norm_residual_backward: lddn smaller than C");
    const bool cols = d_gate || d_scale || d_post_w || d_post_b || d_pre_w || d_pre_b;
    const bool empty = d->samples == 0 || d->rows == 0;
    if (empty && !cols) return 0;
    if (!empty) RDFC_REQUIRE(x && dx && (!h || dh) && stats && (!dn || d->pre) && (!cols || scratch), "rdfc_norm_residual_backward: null pointer");
    RDFC_REQUIRE(((reinterpret_cast<size_t>(stats) & 15) | (reinterpret_cast<size_t>(scratch) & 7)) == 0, "rdfc_norm_residual_backward: stats or scratch is not aligned");
    RDFC_REQUIRE(!d_gate || gate, "rdfc_norm_residual_backward: gradient of a gate that is not there");
    NRArgs p = nr_args(d, x, h, gate, scale, post_w, post_b, pre_w, nullptr, key);
    p.dy = dy;
    p.dn = dn;
    p.lddy = lddy;
    p.lddn = lddn;
    p.dx = dx;
    p.dh = dh;
    p.stats = reinterpret_cast<f32x4 *>(const_cast<float *>(stats));
    p.partial = cols ? scratch : nullptr;
    const int samples = gate ? d->samples : 1;
    NRChunks k = {};
    if (!empty) {
        p.rows = gate ? d->rows : d->rows * d->samples;
        k = bwd_chunks(p.rows, samples, d->C);
        p.chunk = k.chunk;
        const dim3 grid((unsigned)k.nchunk, samples);
        const bool al = row_aligned(x, d->ldx, d->dtype) && row_aligned(h, d->ldh, d->dtype) && row_aligned(dy, lddy, d->dtype) &&
                        row_aligned(dn, lddn, d->dtype) && row_aligned(dx, d->C, d->dtype) && row_aligned(dh, d->C, d->dtype) && d->C % 8 == 0;
        with_layout(d->C, [&](auto lpr, auto vpl) {
            constexpr int L = decltype(lpr)::value, V = decltype(vpl)::value;
            RDFC_DISPATCH(d->dtype, if (al) norm_residual_bwd_kernel<T, L, V, true><<<grid, threads_of(L), 0, (hipStream_t)stream>>>(p);
                          else norm_residual_bwd_kernel<T, L, V, false><<<grid, threads_of(L), 0, (hipStream_t)stream>>>(p));
        });
        RDFC_LAUNCH_CHECK("rdfc_norm_residual_backward");
    }
    if (cols) {
        const NRGrads o = {d_gate, d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b};
        double *sums = reinterpret_cast<double *>(scratch + k.partial);         // (8-byte aligned: partial is a multiple of 4)
        if (!empty)
            norm_residual_sum_kernel<<<dim3(cdiv(4 * d->C, SUM_COLS), samples, k.slices), SUM_COLS * SUM_ROWS, 0, (hipStream_t)stream>>>(scratch, sums, 4 * d->C, k.nchunk);
        norm_residual_grads_kernel<<<cdiv(d->C, 64), 512, 0, (hipStream_t)stream>>>(p, o, sums, samples, k.slices);
        RDFC_LAUNCH_CHECK("rdfc_norm_residual_backward (columns)");
    }
    return 0;
}
