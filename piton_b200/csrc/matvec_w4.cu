// y = x W^T (+ bias) with 4-bit weights W[n, k] = scale[n, k / group] (code[n, k] - zero[n, k / group]), for a few rows x.
//
// The codes are read once (N K / 2 bytes) and bound the product up to about 16 rows, so everything is
// arranged around streaming them.  A warp takes 16 weight rows and a share of the inner dimension in blocks of
// 128; its lanes copy 16 bytes of a row each (cp.async, zero-filled past the row's end) into a queue of their own
// warp, three or more blocks deep, so no warp waits for another before the end.  A code minus its zero point is exact in
// fp16 (the nibble is put into the low bits of 1024's significand), weights are the 16-row side of mma.m16n8k16 and
// the rows of x its 8-column side, and each group's sum is scaled in fp32: no weight is ever rounded.
// 16-bit rows of x enter as they are (scaled by a power of two per row and block); fp32 rows as two
// fp16 halves (22 bits).
#include "decode.cuh"

namespace piton {
namespace decode {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int BLOCK = 128;                  // inner elements of a block: 64 bytes of each of 16 rows
constexpr int QUAD = 80;                    // bytes a row takes in the queue: 64 and 16 that keep reads free of bank conflicts
constexpr int SLOT = 16 * QUAD;

struct MatvecParams {
    const void *x, *scales, *bias;
    const uint8_t *codes, *zeros;
    void *y;
    int64_t rows, inner, outer, sx, sc, ss, sz, sy;
    int32_t group_log2, scale_type, aligned;
};

__device__ __forceinline__ float load_scale(const void *p, int32_t type, int64_t i) {
    if (type == PITON_B200_TYPE_F32) return reinterpret_cast<const float *>(p)[i];
    if (type == PITON_B200_TYPE_F16) return to_float(reinterpret_cast<const __half *>(p)[i]);
    return to_float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(uint32_t packed, float lo, float hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&packed));
    return pack(lo - f.x, hi - f.y);
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// The zero point of a group as the two constants that turn nibbles into code - zero.
struct Zero {
    uint32_t low, high;                     // 1024 + zero and -(64 + zero), twice each
};
__device__ __forceinline__ Zero zero_of(uint32_t z) {
    const __half2 a = __half2half2(__uint2half_rn(1024 + z)), b = __half2half2(__int2half_rn(-(int)(64 + z)));
    return {*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b)};
}
// The eight codes of a word less the zero point, as pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ void weights_of(uint32_t (&h)[4], uint32_t w, const Zero &z) {
    const uint32_t sixteenth = 0x2C002C00u;
    h[0] = hsub2((w & 0x000F000Fu) | 0x64006400u, z.low);                          // 1024 + code
    h[1] = hfma2((w & 0x00F000F0u) | 0x64006400u, sixteenth, z.high);              // 1024 + 16 code
    w >>= 8;
    h[2] = hsub2((w & 0x000F000Fu) | 0x64006400u, z.low);
    h[3] = hfma2((w & 0x00F000F0u) | 0x64006400u, sixteenth, z.high);
}

// NT tiles of 8 rows of x; GROUPS = 128 / group scales of a weight row in a block.
template <typename T, int NT, int GROUPS, int STAGES>
__global__ void __launch_bounds__(THREADS) matvec_w4_kernel(const MatvecParams p) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int CHUNKS = 4 / GROUPS;                      // 32-element chunks of a block that share a scale
    extern __shared__ __align__(16) uint8_t queue[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (8 * NT);
    const int64_t blocks = (p.inner + BLOCK - 1) / BLOCK, bytes = (p.inner + 1) / 2;
    const int mine = blocks > warp ? (int)((blocks - warp + WARPS - 1) / WARPS) : 0;
    const uint8_t *slots = queue + warp * (STAGES * SLOT);
    const uint32_t at0 = (uint32_t)__cvta_generic_to_shared(slots);

    // lane (g, j): bytes 16 j ... 16 j + 15 of a block of weight rows n0 + g and n0 + g + 8
    auto issue = [&](int s) {
        if (s < mine) {
            const int64_t byte = (int64_t)(warp + s * WARPS) * (BLOCK / 2) + 16 * j;
            const int64_t left = bytes - byte;
            const int size = left >= 16 ? 16 : (left > 0 ? (int)left : 0);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t n = n0 + g + 8 * r;
                const int have = n < p.outer ? size : 0;
                const uint8_t *src = p.codes + (have ? n * p.sc + byte : 0);
                const uint32_t dst = at0 + (s % STAGES) * SLOT + (g + 8 * r) * QUAD + 16 * j;
                if (p.aligned) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have) : "memory");
                } else {                                    // rows that do not start on 16 bytes: byte by byte
                    for (int w = 0; w < 4; ++w) {
                        uint32_t word = 0;
                        for (int i = 0; i < 4; ++i)
                            if (4 * w + i < have) word |= (uint32_t)src[4 * w + i] << (8 * i);
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 4 * w), "r"(word) : "memory");
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);

    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;

#pragma unroll 1
    for (int s = 0; s < mine; ++s) {
        const int64_t blk = warp + (int64_t)s * WARPS, k0 = blk * BLOCK;
        // scales and zero points of weight rows n0 + g and n0 + g + 8
        float scale[GROUPS][2];
        Zero zero[GROUPS][2];
#pragma unroll
        for (int q = 0; q < GROUPS; ++q)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t n = n0 + g + 8 * r, group = (k0 >> p.group_log2) + q;
                const bool on = n < p.outer && (group << p.group_log2) < p.inner;
                scale[q][r] = on ? load_scale(p.scales, p.scale_type, n * p.ss + group) : 0.0f;
                zero[q][r] = zero_of(on && p.zeros ? p.zeros[n * p.sz + group] : 8);
            }
        // rows of x: lane (g, j) holds row m0 + 8 t + g, elements 8 j ... 8 j + 7 of each 32-element chunk, scaled by a
        // power of two that brings the block's largest magnitude into [2^14, 2^15)
        uint32_t xh[NT][4][4], xl[SPLIT ? NT : 1][4][4];
        float back[NT][2];                                  // of rows 2 j and 2 j + 1, the columns of the accumulators
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int64_t m = m0 + 8 * t + g;
            const T *x = reinterpret_cast<const T *>(p.x) + (m < p.rows ? m * p.sx : 0);
            float v[4][8], top = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t k = k0 + 32 * c + 8 * j + e;
                    v[c][e] = m < p.rows && k < p.inner ? to_float(x[k]) : 0.0f;
                    top = fmaxf(top, isfinite(v[c][e]) ? fabsf(v[c][e]) : 0.0f);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = top == 0.0f ? 0 : min(max(14 + 127 - (int)(__float_as_uint(top) >> 23), -112), 112);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23), inv = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = v[c][e] * f, hi = v[c][e + 4] * f;
                    xh[t][c][e] = pack(lo, hi);
                    if constexpr (SPLIT) xl[t][c][e] = pack_rest(xh[t][c][e], lo, hi);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) back[t][e] = __shfl_sync(0xffffffffu, inv, 4 * (2 * j + e));
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        const uint32_t at = at0 + (s % STAGES) * SLOT + g * QUAD + 4 * j;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            float part[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[t][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                const int c = q * CHUNKS + i;
                uint32_t w0, w1, h0[4], h1[4];              // word j of chunk c: elements 8 j ... 8 j + 7 of its 32
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0) : "r"(at + 16 * c) : "memory");
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1) : "r"(at + 16 * c + 8 * QUAD) : "memory");
                weights_of(h0, w0, zero[q][0]);
                weights_of(h1, w1, zero[q][1]);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const uint32_t a[4] = {h0[e], h1[e], h0[e + 1], h1[e + 1]};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma(part[t], a, xh[t][c][e], xh[t][c][e + 1]);
                        if constexpr (SPLIT) mma(part[t], a, xl[t][c][e], xl[t][c][e + 1]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] += part[t][e] * back[t][e & 1] * scale[q][e >> 1];
        }
        __syncwarp();                                       // every lane has read the slot that is filled next
        issue(s + STAGES - 1);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float *sums = reinterpret_cast<float *>(queue);         // [WARPS][8 NT rows of x][16 weight rows]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[(warp * 8 * NT + 8 * t + 2 * j + (e & 1)) * 16 + g + 8 * (e >> 1)] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * NT; i += THREADS) {
        const int64_t m = m0 + (i >> 4), n = n0 + (i & 15);
        if (m >= p.rows || n >= p.outer) continue;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += sums[w * 128 * NT + i];
        if (p.bias) sum += to_float(reinterpret_cast<const T *>(p.bias)[n]);
        reinterpret_cast<T *>(p.y)[m * p.sy + n] = from_float<T>(sum);
    }
}

template <typename T, int NT, int GROUPS> int launch(const MatvecParams &p, cudaStream_t s) {
    constexpr int STAGES = 4, SMEM = WARPS * STAGES * SLOT;
    static_assert(WARPS * 128 * NT * 4 <= SMEM && SMEM <= 48 * 1024, "the warps' sums fit the queues");
    const dim3 grid((unsigned)cdiv(p.outer, 16), (unsigned)cdiv(p.rows, 8 * NT));
    matvec_w4_kernel<T, NT, GROUPS, STAGES><<<grid, THREADS, SMEM, s>>>(p);
    return check_launch("matvec_w4");
}

template <typename T, int NT> int launch(const MatvecParams &p, cudaStream_t s) {
    return p.group_log2 == 7 ? launch<T, NT, 1>(p, s) : p.group_log2 == 6 ? launch<T, NT, 2>(p, s) : launch<T, NT, 4>(p, s);
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
    p.group_log2 = a->group == 32 ? 5 : a->group == 64 ? 6 : 7; p.scale_type = a->scale_type;
    p.aligned = a->codes % 16 == 0 && a->stride_codes % 16 == 0;
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        cudaStream_t s = as_stream(stream);
        return a->rows <= 8 ? launch<T, 1>(p, s) : launch<T, 2>(p, s);
    });
}
