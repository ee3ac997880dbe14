// dropout.hip -- elementwise dropout with a mask that is never stored (philox.h).
//
// y[e] = keep(e) ? x[e] * inv : 0.  The backward pass is the same kernel on the cotangent with the same key.
#include "philox.h"

namespace {

constexpr int NT = 256, GPT = 4;      // threads, groups of eight elements per thread

// Groups of eight consecutive elements of the dense order.  VECTOR: every group lies inside a row and is 16-byte aligned in x and y.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(NT) void dropout_kernel(DropArgs d, const T *__restrict__ x, T *__restrict__ y, unsigned long long n, int C, int ldx, int ldy) {
    const unsigned long long seed = d.key ? d.key[0] : d.seed, offset = d.key ? d.key[1] : d.offset;
    const unsigned long long ngroups = (n + 7) >> 3, g0 = (unsigned long long)blockIdx.x * (NT * GPT) + threadIdx.x;
    for (int k = 0; k < GPT; ++k) {
        const unsigned long long q = g0 + k * NT;
        if (q >= ngroups) return;
        unsigned long long row = (q << 3) / (unsigned)C;
        int c = (int)((q << 3) - row * (unsigned)C);
        const unsigned keep = keep8(q << 3, d.threshold, seed, offset);
        for (int i = 0; i < 8 && (q << 3) + i < n; ++i) {
            const float v = Elem<T>::ld(x + row * (unsigned)ldx + c);
            Elem<T>::st(y + row * (unsigned)ldy + c, keep >> i & 1 ? v * d.inv : 0.f);
            if (++c == C) {
                c = 0;
                ++row;
            }
        }
    }
}

// key = {state[0], state[1]}, state[1] += 1: one draw of a device-side generator state
__global__ void dropout_draw_kernel(unsigned long long *state, unsigned long long *key) {
    key[0] = state[0];
    key[1] = state[1]++;
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
    const unsigned long long n = (unsigned long long)P * C, blocks = ((n + 7) / 8 + NT * GPT - 1) / (NT * GPT);
    RDFC_REQUIRE(blocks < (1ull << 31), "rdfc_dropout: %llu elements are too many", n);
    RDFC_DISPATCH(dtype, (dropout_kernel<T, false><<<dim3((unsigned)blocks), NT, 0, (hipStream_t)stream>>>(d, (const T *)x, (T *)y, n, C, ldx, ldy)));
    RDFC_LAUNCH_CHECK("rdfc_dropout");
    return 0;
}

extern "C" int rdfc_dropout_draw(uint64_t *state, uint64_t *key, void *stream) {
    RDFC_REQUIRE(state && key, "rdfc_dropout_draw: null pointer");
    dropout_draw_kernel<<<1, 1, 0, (hipStream_t)stream>>>(reinterpret_cast<unsigned long long *>(state), reinterpret_cast<unsigned long long *>(key));
    RDFC_LAUNCH_CHECK("rdfc_dropout_draw");
    return 0;
}
