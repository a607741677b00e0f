// y = x W^T (+ bias) with 4-bit weights, a scale (and zero point) per group along the inner
// dimension: a warp per output, its lanes along the weight row's bytes.
#include "decode.cuh"

namespace piton {
namespace decode {
namespace {

constexpr int THREADS = 128;

struct MatvecParams {
    const void *x, *scales, *bias;
    const uint8_t *codes, *zeros;
    void *y;
    int64_t rows, inner, outer, sx, sc, ss, sz, sy;
    int32_t group, scale_type;
};

__device__ __forceinline__ float load_scale(const void *p, int32_t type, int64_t i) {
    if (type == PITON_B200_TYPE_F32) return reinterpret_cast<const float *>(p)[i];
    if (type == PITON_B200_TYPE_F16) return to_float(reinterpret_cast<const __half *>(p)[i]);
    return to_float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) matvec_w4_kernel(const MatvecParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), m = blockIdx.y;
    if (n >= p.outer) return;
    const T *x = reinterpret_cast<const T *>(p.x) + m * p.sx;
    const uint8_t *w = p.codes + n * p.sc;
    float acc = 0.0f;
    for (int64_t k = 2 * lane; k < p.inner; k += 64) {
        const int64_t g = k / p.group;                               // even k and group: both halves are in one group
        const uint8_t c = w[k >> 1];
        const float zero = p.zeros ? (float)p.zeros[n * p.sz + g] : 8.0f;
        float part = to_float(x[k]) * ((float)(c & 15) - zero);
        if (k + 1 < p.inner) part += to_float(x[k + 1]) * ((float)(c >> 4) - zero);
        acc += part * load_scale(p.scales, p.scale_type, n * p.ss + g);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) {
        if (p.bias) acc += to_float(reinterpret_cast<const T *>(p.bias)[n]);
        reinterpret_cast<T *>(p.y)[m * p.sy + n] = from_float<T>(acc);
    }
}

}  // namespace
}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

extern "C" int piton_b200_matvec_w4(const piton_matvec_w4_args *a, void *stream) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->scale_type >= PITON_B200_TYPE_F32 && a->scale_type <= PITON_B200_TYPE_BF16, "unknown scale type %d",
                  a->scale_type);
    PITON_REQUIRE(a->rows >= 0 && a->inner >= 0 && a->outer >= 0, "bad shape");
    PITON_REQUIRE(a->rows <= 65535 && a->outer < (1ll << 31) && a->inner < (1ll << 31), "rows, inner or outer too large");
    if (a->group != 32 && a->group != 64 && a->group != 128)
        return set_error(PITON_B200_ENOTSUP, "group %d (32, 64, 128)", a->group);
    if (a->rows == 0 || a->outer == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->y && (a->inner == 0 || (a->x && a->codes && a->scales)), "NULL pointer");
    MatvecParams p;
    p.x = reinterpret_cast<const void *>(a->x);
    p.codes = reinterpret_cast<const uint8_t *>(a->codes);
    p.scales = reinterpret_cast<const void *>(a->scales);
    p.zeros = reinterpret_cast<const uint8_t *>(a->zeros);
    p.bias = reinterpret_cast<const void *>(a->bias);
    p.y = reinterpret_cast<void *>(a->y);
    p.rows = a->rows; p.inner = a->inner; p.outer = a->outer;
    p.sx = a->stride_x; p.sc = a->stride_codes; p.ss = a->stride_scales; p.sz = a->stride_zeros; p.sy = a->stride_y;
    p.group = a->group; p.scale_type = a->scale_type;
    const dim3 grid((unsigned)cdiv(a->outer, THREADS / 32), (unsigned)a->rows);
    return with_type(a->type, [&](auto t) {
        matvec_w4_kernel<decltype(t)><<<grid, THREADS, 0, as_stream(stream)>>>(p);
        return check_launch("matvec_w4");
    });
}
