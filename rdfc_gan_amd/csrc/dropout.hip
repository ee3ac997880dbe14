// dropout.hip -- elementwise dropout with a mask that is never stored (philox.h).
//
// y[e] = keep(e) ? x[e] * inv : 0.  The backward pass is the same kernel on the cotangent with the same key.
//
// HBM bounds it: 16x228x304x64 in bf16 takes 50 us a pass, 284 MB at 5.6 TB/s (x + 1 over 2 GB reaches 6.2 on the same card, and a pass that moved its
// elements one by one took 160).  A generator call is 18 wide multiplications and about 110 other vector instructions for eight elements, by
// count some 40 us of the same pass on all SIMDs, under the loads: 32 bits an element would take twice that and bind.
// Small maps are bound by the launch: 8x15x19x512 in f16 3 us.
#include "philox.h"

namespace {

constexpr int NT = 256;

template <typename T> struct Eight {               // eight consecutive elements: one 16-byte vector, two in f32
    static constexpr int NV = 8 / Elem<T>::VEC;
    Vec16<T> v[NV];
    __device__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].load(p + i * Elem<T>::VEC);
    }
    __device__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].store(p + i * Elem<T>::VEC);
    }
    __device__ float get(int i) const { return v[i / Elem<T>::VEC].get(i % Elem<T>::VEC); }
    __device__ void set(int i, float f) { v[i / Elem<T>::VEC].set(i % Elem<T>::VEC, f); }
};

// Groups of eight consecutive elements of the dense order, GPT per thread, all their loads in flight before the first mask is drawn.
//   FLAT     x and y are dense: a group is at 8 q in both
//   ROWS     C is a multiple of 8 and every row 16-byte aligned: a group lies inside a row
//   ANY      everything else: element by element
// WIDE: element indexes of 64 bits (the division by C costs about three times a 32-bit one)
enum { FLAT, ROWS, ANY };
template <typename T, int HOW, int GPT, bool WIDE>
__global__ __launch_bounds__(NT) void dropout_kernel(DropArgs d, const T *__restrict__ x, T *__restrict__ y, unsigned long long n, int C, int ldx, int ldy) {
    using I = typename std::conditional<WIDE, unsigned long long, unsigned>::type;
    const unsigned long long seed = d.key ? d.key[0] : d.seed, offset = d.key ? d.key[1] : d.offset;
    const I ngroups = (I)((n + 7) >> 3), g0 = (I)blockIdx.x * (NT * GPT) + threadIdx.x;
    if constexpr (HOW != ANY) {
        Eight<T> v[GPT];
        unsigned long long dst[GPT];
#pragma unroll
        for (int k = 0; k < GPT; ++k) {
            const I q = g0 + k * NT;
            if (q < ngroups) {
                unsigned long long src = (unsigned long long)q << 3;
                dst[k] = src;
                if constexpr (HOW == ROWS) {
                    const I row = q / (unsigned)(C >> 3);
                    const unsigned c = (unsigned)(q - row * (unsigned)(C >> 3)) << 3;
                    src = (unsigned long long)row * (unsigned)ldx + c;
                    dst[k] = (unsigned long long)row * (unsigned)ldy + c;
                }
                v[k].load(x + src);
            }
        }
#pragma unroll
        for (int k = 0; k < GPT; ++k) {
            const I q = g0 + k * NT;
            if (q >= ngroups) break;
            const u32x4 w = philox(q, seed, offset);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k].set(i, word16(w, i) >= d.threshold ? v[k].get(i) * d.inv : 0.f);
            v[k].store(y + dst[k]);
        }
    } else {
        static_assert(HOW != ANY || GPT == 1, "one group a thread where elements move one by one");
        if (g0 >= ngroups) return;
        const unsigned long long e0 = (unsigned long long)g0 << 3;
        unsigned long long row;
        unsigned c;
        if (WIDE) row = e0 / (unsigned)C;
        else row = (unsigned)e0 / (unsigned)C;
        c = (unsigned)(e0 - row * (unsigned)C);
        const int m = n - e0 < 8 ? (int)(n - e0) : 8;
        float v[8];
        unsigned long long dst[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dst[i] = row * (unsigned)ldy + c;
            v[i] = i < m ? Elem<T>::ld(x + row * (unsigned)ldx + c) : 0.f;
            if (++c == (unsigned)C) {
                c = 0;
                ++row;
            }
        }
        const u32x4 w = philox(g0, seed, offset);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < m) Elem<T>::st(y + dst[i], word16(w, i) >= d.threshold ? v[i] * d.inv : 0.f);
    }
}

// key = {state[0], state[1]}, state[1] += 1: one draw of a device-side generator state (draws on several streams at once get keys of their own)
__global__ void dropout_draw_kernel(unsigned long long *state, unsigned long long *key) {
    key[0] = state[0];
    key[1] = atomicAdd(state + 1, 1ull);
}

}  // namespace

extern "C" int rdfc_dropout(const void *x, void *y, int64_t P, int C, int ldx, int ldy, int dtype, int threshold, uint64_t seed, uint64_t offset,
                            const uint64_t *key, void *stream) {
    RDFC_REQUIRE(rdfc_dtype_ok(dtype), "rdfc_dropout: unsupported dtype %d", dtype);
    RDFC_REQUIRE(P >= 0 && C > 0 && ldx >= C && ldy >= C, "rdfc_dropout: bad sizes P=%lld C=%d ldx=%d ldy=%d", (long long)P, C, ldx, ldy);
    DropArgs d;
    RDFC_REQUIRE(drop_args(d, threshold, seed, offset, key), "rdfc_dropout: threshold %d is not in [0, 65536]", threshold);
    if (P == 0) return 0;
    RDFC_REQUIRE(x && y, "rdfc_dropout: null map");
    const unsigned long long n = (unsigned long long)P * C, groups = (n + 7) / 8;
    const int vec = rdfc_vec(dtype);
    const bool al = ((reinterpret_cast<size_t>(x) | reinterpret_cast<size_t>(y)) & 15) == 0;
    // (a dense map with a last group that is not whole goes element by element)
    const int how = al && ldx == C && ldy == C && n % 8 == 0 ? FLAT : al && C % 8 == 0 && ldx % vec == 0 && ldy % vec == 0 ? ROWS : ANY;
    const int gpt = how == ANY ? 1 : groups >= 256 * 2048 ? 4 : 1;
    const unsigned long long blocks = (groups + NT * gpt - 1) / (NT * gpt);
    const bool wide = n + 8ull * NT * gpt >= 1ull << 32;
    RDFC_REQUIRE(blocks < (1ull << 31), "rdfc_dropout: %llu elements are too many", n);
    auto go = [&](auto h, auto g, auto w) {
        constexpr int H = decltype(h)::value, G = decltype(g)::value;
        constexpr bool W = decltype(w)::value;
        RDFC_DISPATCH(dtype, (dropout_kernel<T, H, G, W><<<dim3((unsigned)blocks), NT, 0, (hipStream_t)stream>>>(d, (const T *)x, (T *)y, n, C, ldx, ldy)));
    };
    auto pick = [&](auto w) {
        if (how == FLAT) gpt == 4 ? go(std::integral_constant<int, FLAT>{}, std::integral_constant<int, 4>{}, w) : go(std::integral_constant<int, FLAT>{}, std::integral_constant<int, 1>{}, w);
        else if (how == ROWS) gpt == 4 ? go(std::integral_constant<int, ROWS>{}, std::integral_constant<int, 4>{}, w) : go(std::integral_constant<int, ROWS>{}, std::integral_constant<int, 1>{}, w);
        else go(std::integral_constant<int, ANY>{}, std::integral_constant<int, 1>{}, w);
    };
    if (wide) pick(std::true_type{});
    else pick(std::false_type{});
    RDFC_LAUNCH_CHECK("rdfc_dropout");
    return 0;
}

extern "C" int rdfc_dropout_draw(uint64_t *state, uint64_t *key, void *stream) {
    RDFC_REQUIRE(state && key, "rdfc_dropout_draw: null pointer");
    dropout_draw_kernel<<<1, 1, 0, (hipStream_t)stream>>>(reinterpret_cast<unsigned long long *>(state), reinterpret_cast<unsigned long long *>(key));
    RDFC_LAUNCH_CHECK("rdfc_dropout_draw");
    return 0;
}
