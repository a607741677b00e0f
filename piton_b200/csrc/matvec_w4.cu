// y = x W^T (+ bias) with 4-bit weights W[n, k] = scale[n, k / group] (code[n, k] - zero[n, k / group]), for a few rows x.
//
// The codes are read once (N K / 2 bytes) and bound the product up to about 16 rows, so everything is
// arranged around streaming them with few instructions a byte.  A warp takes 16 R weight rows in steps of 256 inner
// elements (128 bytes of a row), copied with cp.async into a queue of its own, so no warp waits for another while it
// streams.  Codes less their zero points are the 16-row side of mma.m16n8k16 and the rows of x its 8-column side.  Both are
// exact: codes become 16-bit floats by a mask and one subtraction for two of them (9 instructions per 8 codes in fp16, 11 in bf16), x stays as
// it is, and fp32 is the sum of three bf16 elements of 8 bits of significand each.  So only the fp32 sums are rounded, and something large
// in x that meets weights of zero costs the rest nothing.  (Sums in integers over x in fixed point take 3 instructions per 8
// codes and 28.0 us for one row of 28000 x 8192 where this takes 38, but lose what a row's small elements have below 2^-16 of a large one;
// taking zero * sum(x) off the sum of code * x loses what the two have in common.)  The group's scale is applied in fp32, two outputs an
// instruction.  x is put into the order of the fragments by every CTA, or once by a small kernel into a workspace, from where a
// CTA copies its share.
//
// A matrix with many rows gives every warp rows of its own (warps along the rows); one with few splits each
// CTA's inner dimension over its eight warps (warps along the inner dimension).  Either way a cluster of CTAs
// may split the inner dimension further, and adds its parts through distributed shared memory in a fixed order.
//
// Measured: 28000 x 8192, groups of 128: 1 row, bf16 38 us (3.1 TB/s), fp16 35.5; 8 rows of bf16, groups of 32 with zero points 70;
// 16 rows of fp32, groups of 64 with zero points 112. 4096 x 4096: 1 row, bf16 6.0 us, 16 rows 9.9; fp32, 8 rows 12.6, 16 rows 13.7; 32768 x
// 8192, bf16, 16 rows 54 us (2.6 TB/s). Rows of codes on any byte: 4096 x 4098 9.0 us, copies of 4 bytes a lane where whole rows take
// 16. A call has 4 to 5 us that do not depend on the matrix (launches, x, the cluster's sums). One row of 28000 x 8192 issues in 52 % of an
// SM's cycles and reads at 36 % of DRAM's, with 220 CTAs for 296 places; 16 rows of 32768 x 8192 in 47 %, waiting for the tensor pipe.
#include <cooperative_groups.h>

#include <type_traits>

#include "decode.cuh"

namespace piton {
namespace decode {
namespace {

namespace cg = cooperative_groups;

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int BLOCK = 128;                  // inner elements: 64 bytes of a weight row
constexpr int LINE = 128;                   // bytes of a weight row in a step: two blocks
constexpr int MAX_PARTS = 8;

struct MatvecParams {
    const void *x, *scales, *bias;
    const uint8_t *codes, *zeros;
    void *y;
    int64_t rows, outer, sx, sc, ss, sz, sy;
    int32_t inner, group_log2, scale_type, codes_align, x_aligned;
    uint8_t *laid;                          // x laid out in the workspace, or null: every CTA lays out what it needs
    int32_t span, phase;                    // steps of a CTA's part, and of what shared memory holds of x at a time
};

// c = a b + c, or a b: fp16 operands for rows of fp16, bf16 operands for the other types.
template <typename T, bool FIRST> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>) {
        if constexpr (FIRST)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        if constexpr (FIRST)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// (w & mask) | bits.
template <uint32_t MASK, uint32_t BITS> __device__ __forceinline__ uint32_t masked(uint32_t w) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "n"(MASK), "r"(BITS));
    return d;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// A weight row's zero point, made ready for its codes, and eight codes less the zero point: pairs of elements 0 and 4, 1 and 5,
// 2 and 6, 3 and 7 of a word. A masked code is the low end of the significand of 1024 (fp16, where the codes four bits up
// count 16) or of 128 (bf16); taking 1024 + zero or 128 + zero from it is exact. In bf16 that holds for zero points up to 127;
// what larger ones are more than their low seven bits is taken off afterwards. There a code counts 2^-8, so that sums of elements near the
// type's largest stay in range until the scale is applied; the outputs are multiplied by UP.
template <typename T> struct Zero {
    static constexpr float UP = 256.0f;
    uint32_t low;                                                       // -(128 + zero) / 256, twice
    // byte i of a word of zero points below 128
    __device__ __forceinline__ Zero(uint32_t z, int i) { low = __byte_perm(z, 0xBF, 0x4040 | 0x101 * i); }
    __device__ __forceinline__ void less(uint32_t (&a)[4], uint32_t w) const {
        constexpr uint32_t DOWN = 0x3B803B80u;                          // 1 / 256
        a[0] = fma_bf16x2(masked<0x000F000Fu, 0x43004300u>(w), DOWN, low);
        a[1] = fma_bf16x2(masked<0x000F000Fu, 0x43004300u>(w >> 4), DOWN, low);
        a[2] = fma_bf16x2(masked<0x000F000Fu, 0x43004300u>(w >> 8), DOWN, low);
        a[3] = fma_bf16x2(masked<0x000F000Fu, 0x43004300u>(w >> 12), DOWN, low);
    }
};
template <> struct Zero<__half> {
    static constexpr float UP = 1.0f;
    uint32_t low, low16;                                                // 1024 + zero; -(64 + zero), twice
    __device__ __forceinline__ Zero(uint32_t z, int i) {
        low = __byte_perm(z, 0x64, 0x4040 | 0x101 * i);
        low16 = sub_f16x2(0x63806380u, low);                            // 960 - (1024 + zero)
    }
    __device__ __forceinline__ void less(uint32_t (&a)[4], uint32_t w) const {
        constexpr uint32_t SIXTEENTH = 0x2C002C00u;
        a[0] = sub_f16x2(masked<0x000F000Fu, 0x64006400u>(w), low);
        a[1] = fma_f16x2(masked<0x00F000F0u, 0x64006400u>(w), SIXTEENTH, low16);
        a[2] = sub_f16x2(masked<0x000F000Fu, 0x64006400u>(w >> 8), low);
        a[3] = fma_f16x2(masked<0x00F000F0u, 0x64006400u>(w >> 8), SIXTEENTH, low16);
    }
};

__device__ __forceinline__ uint4 load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// Two floats in one 64-bit register, and the instructions that take two at a time: half as many to issue.
typedef unsigned long long pair;
__device__ __forceinline__ pair both(float a, float b) {
    pair d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) {
    pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// NT tiles of 8 rows of x, R tiles of 16 weight rows a warp, GROUPS = 128 / group scales of a weight row in a block.
template <typename T, int NT, int R, int GROUPS> struct Shape {
    // Of each group's 32 WORDS elements in a block lane j takes the 8 WORDS from 8 WORDS j on: WORDS words of codes.
    static constexpr int WORDS = 4 / GROUPS;
    // Two stages (three: one row of 28000 x 8192, bf16, 39.5 us, two 37.8; 16 rows of 32768 x 8192 64 and 54; 4096 x 4096 6.0 either way)
    static constexpr int SLOT = 16 * R * LINE + 128, STAGES = 2, QUEUES = WARPS * STAGES * SLOT;
    static constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;               // of x
    static constexpr int SUMS = 8 * NT * 16 * R;                        // outputs of a warp's tile
    // x in shared memory, per row: 16 bytes for every 8 elements of a piece; the padding puts rows that are read together into
    // different banks
    static constexpr int STEP_BYTES = 512 * PIECES;                     // a row's part of a step
    __host__ __device__ static constexpr int pitch(int steps) { return steps * STEP_BYTES + 64; }
    // shared memory: queues (in the end the warps' sums), x
    static_assert(WARPS * SUMS * 4 <= QUEUES, "the sums fit");
    static int64_t smem(int64_t rows, int64_t steps) { return QUEUES + rows * pitch((int)steps); }
};

// Lays out `steps` steps from step0 on of the rows m0 ...: per row and block 16 units of 8 elements, unit 4 c + j for word c of lane
// j (word w of group q: c = q WORDS + w), which faces elements 32 WORDS q + 8 WORDS j + 8 w ... of the block. A unit's elements lie as the
// codes of a word come out: 0, 4, 1, 5, 2, 6, 3, 7. An fp32 element is the sum of three bf16 ones, its upper, middle and lower 8 bits of
// significand, exactly (but for what lies below 2^-133); they lie in 16 bytes a piece.
template <typename T, int WORDS>
__device__ __forceinline__ void lay_out(const MatvecParams &p, int64_t m0, int x_rows, int step0, int steps, uint8_t *to, int64_t pitch) {
    constexpr int PIECES = sizeof(T) == 4 ? 3 : 1, AT_ONCE = PIECES == 1 ? 4 : 2;    // units that a thread has on their way
    const int count = 2 * steps, units = x_rows * count * 16;
    for (int u0 = threadIdx.x; u0 < units; u0 += AT_ONCE * THREADS) {
        T v[AT_ONCE][8];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const int u = u0 + n * THREADS, unit = u & 15, c = unit >> 2, b = (u >> 4) % count, m = (u >> 4) / count;
            const int k = (2 * step0 + b) * BLOCK + c / WORDS * (32 * WORDS) + 8 * WORDS * (unit & 3) + 8 * (c % WORDS);
            const bool in = u < units;
            const T *src = reinterpret_cast<const T *>(p.x) + (m0 + (in ? m : 0)) * p.sx + k;
            if (in && k + 8 <= p.inner && p.x_aligned) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(v[n])[i] = reinterpret_cast<const uint4 *>(src)[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[n][i] = in && k + i < p.inner ? src[i] : from_float<T>(0.0f);
            }
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            const int u = u0 + n * THREADS, unit = u & 15, b = (u >> 4) % count, m = (u >> 4) / count;
            if (u >= units) break;
            uint4 *at = reinterpret_cast<uint4 *>(to + m * pitch + (b * 16 + unit) * (16 * PIECES));
            if constexpr (PIECES == 1) {
                const uint4 r = *reinterpret_cast<const uint4 *>(v[n]);
                at[0] = make_uint4(__byte_perm(r.x, r.z, 0x5410), __byte_perm(r.x, r.z, 0x7632), __byte_perm(r.y, r.w, 0x5410), __byte_perm(r.y, r.w, 0x7632));
            } else {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = to_float(v[n][i]);
#pragma unroll
                for (int piece = 0; piece < PIECES; ++piece) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = __byte_perm(__float_as_uint(f[i]), __float_as_uint(f[4 + i]), 0x7632);     // the upper halves
                    at[piece] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int i = 0; i < 8; ++i)                          // an infinity has no rest, of a NaN a NaN is left
                        f[i] = fabsf(f[i]) == INFINITY ? 0.0f : f[i] - __uint_as_float(__float_as_uint(f[i]) & 0xFFFF0000u);
                }
            }
        }
    }
}

// Rows of fp32 laid out once for all CTAs, which would otherwise split them again for every 16 or 256 weight rows: a thread a unit.
template <typename T, int WORDS> __global__ void __launch_bounds__(THREADS) matvec_w4_layout_kernel(const MatvecParams p, int all_steps) {
    const int step = blockIdx.x * 8, m = blockIdx.y;
    const int64_t pitch = all_steps * (512 * (sizeof(T) == 4 ? 3 : 1));
    lay_out<T, WORDS>(p, m, 1, step, min(8, all_steps - step), p.laid + m * pitch + step * (pitch / all_steps), pitch);
    asm volatile("griddepcontrol.launch_dependents;");
}

// ALONG_K: the CTA's warps share 16 R weight rows and split the inner dimension; otherwise each has rows of its own.
template <typename T, int NT, int R, int GROUPS, bool ALONG_K, bool BYTES>
__global__ void __launch_bounds__(THREADS, 2) matvec_w4_kernel(const MatvecParams p) {
    using S = Shape<T, NT, R, GROUPS>;
    constexpr int WORDS = S::WORDS, STAGES = S::STAGES, STRIDE = ALONG_K ? WARPS : 1, PIECES = S::PIECES, STEP = 2 * BLOCK;
    extern __shared__ __align__(128) uint8_t queue[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int64_t m0 = (int64_t)blockIdx.y * (8 * NT);
    const int x_rows = (int)min((int64_t)(8 * NT), p.rows - m0);
    const int step0 = part * p.span, steps = max(min(p.span, (p.inner + STEP - 1) / STEP - step0), 0);   // this CTA's
    const int own0 = ALONG_K ? warp : 0, own = steps > own0 ? (steps - own0 + STRIDE - 1) / STRIDE : 0;  // this warp's

    // A warp's weight rows; the last ones are moved back to end with the matrix, so that all 16 R exist (R > 1 only where outer
    // >= 16 R); rows that are computed twice come out the same both times.
    const int64_t tile = (int64_t)(blockIdx.x / parts) * (ALONG_K ? 1 : WARPS) + (ALONG_K ? 0 : warp);
    const int64_t n0 = min(tile * (16 * R), max(p.outer - 16 * R, (int64_t)0));
    const int rows = (int)min((int64_t)(16 * R), p.outer - n0);
    // the weight row (and that + 8) of a tile that fragment row g is: rows that are read together lie in different banks
    const int row = WORDS == 4 ? (g & 1) << 2 | g >> 1 : WORDS == 2 ? (g & 3) << 1 | g >> 2 : g;

    // ---- the queue: in a slot, row r's 128 bytes lie at 128 r, its 16-byte pieces exchanged by r % 8. Rows that do not start on 4
    // bytes are copied from the word before on, and put right as they are read; their last words follow the rows ----
    const uint32_t at0 = (uint32_t)__cvta_generic_to_shared(queue) + warp * (STAGES * S::SLOT);
    const uint8_t *codes = p.codes + n0 * p.sc + (int64_t)(step0 + own0) * LINE;
    const uint32_t copy_at = (lane >> 3) * LINE + ((lane & 7) ^ (lane >> 3)) * 16;
    uint32_t fill = at0;
    int issued = 0;
    auto issue = [&]() {
        if (issued < own) {
            const bool whole = (step0 + own0 + issued * STRIDE + 1) * STEP <= p.inner;
            if (whole && p.codes_align == 16) {                         // 4 rows a copy, 8 lanes each
                const uint8_t *src = codes + (lane >> 3) * p.sc + 16 * (lane & 7);
                const uint32_t dst[2] = {fill + copy_at, (fill + copy_at) ^ 64};     // rows r and r + 4: pieces exchanged by 4
#pragma unroll
                for (int i = 0; i < 4 * R; ++i) {
                    if (R > 1 || 4 * i + (lane >> 3) < rows) copy_async<16>(dst[i & 1] + 512 * i, src);
                    src += 4 * p.sc;
                }
            } else if (whole && p.codes_align == 4) {                   // a row a copy
                const uint8_t *src = codes + 4 * lane;
#pragma unroll 8
                for (int r = 0; r < 16 * R; ++r) {
                    if (R > 1 || r < rows) copy_async<4>(fill + 128 * r + ((lane >> 2) ^ (r & 7)) * 16 + 4 * (lane & 3), src);
                    src += p.sc;
                }
            } else {                                                    // the last step, or rows that are not aligned: words that hold a byte of the row
                const uint8_t *src = codes;
                const int64_t left = (p.inner + 1) / 2 - (int64_t)(step0 + own0 + issued * STRIDE) * LINE;
#pragma unroll 4
                for (int r = 0; r < rows; ++r) {
                    const int before = (int)(reinterpret_cast<uintptr_t>(src) & 3);
                    if (4 * lane - before < left) copy_async<4>(fill + 128 * r + ((lane >> 2) ^ (r & 7)) * 16 + 4 * (lane & 3), src - before + 4 * lane);
                    src += p.sc;
                }
                src = codes + lane * p.sc;
                const int before = (int)(reinterpret_cast<uintptr_t>(src) & 3);
                if (before && lane < rows && LINE - before < left) copy_async<4>(fill + 16 * R * LINE + 4 * lane, src - before + LINE);
            }
            codes += STRIDE * LINE;
            ++issued;
            fill = fill == at0 + (STAGES - 1) * S::SLOT ? at0 : fill + S::SLOT;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue();

    // ---- scales and zero points, a load ahead: lane (g, j) holds those of its 2 R weight rows for one group in four: with
    // group 128 the four groups of two steps, with 64 those of a step, with 32 those of a block (two loads a step); zero points
    // of the rows share a word, a byte each ----
    constexpr int LOADS = GROUPS == 4 ? 2 : 1, AHEAD = GROUPS == 1 ? 2 : 1;    // loads in a step, steps of a load
    uint32_t scale[LOADS][2 * R], scale_next[LOADS][2 * R], zeros[LOADS], zeros_next[LOADS];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) zeros[l] = zeros_next[l] = 0x08080808u;
    const int groups = (p.inner + (1 << p.group_log2) - 1) >> p.group_log2;
    const int64_t scale_row = (n0 + row) * p.ss, zero_row = (n0 + row) * p.sz;
    auto fetch = [&](int turn) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const int step = step0 + own0 + (turn + (GROUPS == 1 ? j >> 1 : 0)) * STRIDE;
            const int group = step * (2 * GROUPS) + (GROUPS == 1 ? j & 1 : 4 * l + j);
            const bool in = turn + (GROUPS == 1 ? j >> 1 : 0) < own && group < groups;
            if (p.scale_type == PITON_B200_TYPE_F32) {
                const uint32_t *at = reinterpret_cast<const uint32_t *>(p.scales) + scale_row + group;
#pragma unroll
                for (int h = 0; h < 2 * R; ++h) scale_next[l][h] = in && row + 8 * h < rows ? at[8 * h * p.ss] : 0;
            } else {
                const uint16_t *at = reinterpret_cast<const uint16_t *>(p.scales) + scale_row + group;
#pragma unroll
                for (int h = 0; h < 2 * R; ++h) scale_next[l][h] = in && row + 8 * h < rows ? at[8 * h * p.ss] : 0;
            }
            if (p.zeros) {
                const uint8_t *at = p.zeros + zero_row + group;
                zeros_next[l] = 0;
#pragma unroll
                for (int h = 0; h < 2 * R; ++h) zeros_next[l] |= (in && row + 8 * h < rows ? (uint32_t)at[8 * h * p.sz] : 0u) << (8 * h);
            }
        }
    };
    fetch(0);

    // ---- x in shared memory; rows of x past the last read the last: a column of the product depends on its own row alone ----
    uint8_t *xs = queue + S::QUEUES;
    uint32_t x_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
        x_at[t] = (uint32_t)__cvta_generic_to_shared(xs) + min(8 * t + g, x_rows - 1) * S::pitch(p.phase) + 16 * PIECES * j;

    pair acc[R][NT][2];                                                 // weight rows row + 8 h, rows 2 j and 2 j + 1 of x
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[r][t][h] = 0;

    uint32_t before = 0;                                                // a byte each: the bits before rows row, row + 8, ... in their first words
#pragma unroll
    for (int h = 0; h < 2 * R; ++h) before |= (uint32_t)(reinterpret_cast<uintptr_t>(p.codes + (n0 + row + 8 * h) * p.sc) & 3) << (8 * h + 3);
    uint32_t slot = at0;
    int turn = 0;
#pragma unroll 1
    for (int phase0 = 0; phase0 < steps; phase0 += p.phase) {
        if (phase0) __syncthreads();                                    // the last phase's x has been read
        const int count = min(p.phase, steps - phase0);
        if (p.laid) {                                                   // 16 bytes at a time, as they lie in the workspace
            const int64_t pitch = (int64_t)((p.inner + STEP - 1) / STEP) * S::STEP_BYTES;
            if (phase0 == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
            const uint8_t *src = p.laid + m0 * pitch + (int64_t)(step0 + phase0) * S::STEP_BYTES;
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(xs);
            for (int m = warp; m < x_rows; m += WARPS)
#pragma unroll 4
                for (int i = 16 * lane; i < count * S::STEP_BYTES; i += 512) copy_async<16>(to + m * S::pitch(p.phase) + i, src + m * pitch + i);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        } else {
            lay_out<T, WORDS>(p, m0, x_rows, step0 + phase0, count, xs, S::pitch(p.phase));
        }
        __syncthreads();
        const int phase_end = phase0 + count;
#pragma unroll 1
        for (; own0 + turn * STRIDE < phase_end; ++turn) {
            if (AHEAD == 1 || !(turn & 1)) {
#pragma unroll
                for (int l = 0; l < LOADS; ++l) {
                    zeros[l] = zeros_next[l];
                    if (p.scale_type == PITON_B200_TYPE_F32) {
#pragma unroll
                        for (int h = 0; h < 2 * R; ++h) scale[l][h] = scale_next[l][h];
                    } else if (p.scale_type == PITON_B200_TYPE_BF16) {
#pragma unroll
                        for (int h = 0; h < 2 * R; ++h) scale[l][h] = scale_next[l][h] << 16;
                    } else {
#pragma unroll
                        for (int h = 0; h < 2 * R; ++h) scale[l][h] = __float_as_uint(__half2float(__ushort_as_half((uint16_t)scale_next[l][h])));
                    }
                }
                fetch(turn + AHEAD);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();                                               // every lane's copies, and the slot that is filled next has been read
            issue();
            const int b0 = 2 * (own0 + turn * STRIDE - phase0);         // block of the phase
            const uint32_t wat = slot + row * LINE + (((WORDS * j >> 2) ^ (row & 7)) * 16) + (4 * WORDS * j & 15);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) {
                    constexpr int LAST = LOADS - 1;
                    const int load = GROUPS == 4 ? b & LAST : 0;
                    const int from = (lane & ~3) | (GROUPS == 1 ? (turn & 1) * 2 + b : GROUPS == 2 ? 2 * b + q : q);
                    const uint32_t z = __shfl_sync(0xffffffffu, zeros[load], from);
                    // WORDS words of codes from byte 64 b + 16 WORDS q + 4 WORDS j of the rows 16 r + row + 8 h
                    uint32_t w[R][2][WORDS];
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            load_words(w[r][h], (wat ^ (64 * b + 16 * WORDS * q)) + (16 * r + 8 * h) * LINE);
                            if constexpr (BYTES) {
                                const int next = 16 * b + 4 * WORDS * q + WORDS * j + WORDS;    // the word after them
                                uint32_t v[1];
                                load_words(v, next == LINE / 4 ? slot + 16 * R * LINE + 4 * (16 * r + row + 8 * h)
                                                               : slot + (16 * r + row + 8 * h) * LINE + ((next >> 2) ^ (row & 7)) * 16 + 4 * (next & 3));
#pragma unroll
                                for (int i = 0; i < WORDS; ++i) w[r][h][i] = __funnelshift_r(w[r][h][i], i + 1 < WORDS ? w[r][h][i + 1] : v[0], before >> (8 * (2 * r + h)));
                            }
                        }
                    const uint32_t z7 = std::is_same_v<T, __half> ? z : z & 0x7F7F7F7Fu;
                    const Zero<T> zero[4] = {{z7, 0}, {z7, 1}, {z7, 2}, {z7, 3}};
                    // the first piece of x, and the smaller ones by themselves, whose sums would be rounded to the first's
                    float sum[R][NT][4], small[PIECES > 1 ? R : 1][NT][4];
#pragma unroll
                    for (int i = 0; i < WORDS; ++i) {
                        uint4 x[NT][PIECES];
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int piece = 0; piece < PIECES; ++piece)
                                x[t][piece] = load16(x_at[t] + (b0 + b) * (256 * PIECES) + (q * WORDS + i) * (64 * PIECES) + 16 * piece);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            uint32_t a0[4], a1[4];
                            zero[2 * r].less(a0, w[r][0][i]);
                            zero[2 * r + 1].less(a1, w[r][1][i]);
                            const uint32_t low[4] = {a0[0], a1[0], a0[1], a1[1]}, high[4] = {a0[2], a1[2], a0[3], a1[3]};
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                if (i == 0) mma<T, true>(sum[r][t], low, x[t][0].x, x[t][0].y);
                                else mma<T, false>(sum[r][t], low, x[t][0].x, x[t][0].y);
                                mma<T, false>(sum[r][t], high, x[t][0].z, x[t][0].w);
                                if constexpr (PIECES > 1) {
                                    if (i == 0) mma<T, true>(small[r][t], low, x[t][2].x, x[t][2].y);
                                    else mma<T, false>(small[r][t], low, x[t][2].x, x[t][2].y);
                                    mma<T, false>(small[r][t], high, x[t][2].z, x[t][2].w);
                                    mma<T, false>(small[r][t], low, x[t][1].x, x[t][1].y);
                                    mma<T, false>(small[r][t], high, x[t][1].z, x[t][1].w);
                                }
                            }
                        }
                    }
                    if constexpr (!std::is_same_v<T, __half>) {
                        if (__any_sync(0xffffffffu, z & 0x80808080u)) {  // zero points from 128 on: what they are more than their low seven bits
#pragma unroll
                            for (int i = 0; i < WORDS; ++i)
#pragma unroll
                                for (int t = 0; t < NT; ++t)
#pragma unroll
                                    for (int piece = 0; piece < PIECES; ++piece) {
                                        const uint4 x = load16(x_at[t] + (b0 + b) * (256 * PIECES) + (q * WORDS + i) * (64 * PIECES) + 16 * piece);
#pragma unroll
                                        for (int r = 0; r < R; ++r) {
                                            const uint32_t d0 = z >> (16 * r + 7) & 1 ? 0xBF00BF00u : 0u, d1 = z >> (16 * r + 15) & 1 ? 0xBF00BF00u : 0u;
                                            const uint32_t a[4] = {d0, d1, d0, d1};                     // -128 / 256 or 0
                                            mma<T, false>(piece ? small[r][t] : sum[r][t], a, x.x, x.y);
                                            mma<T, false>(piece ? small[r][t] : sum[r][t], a, x.z, x.w);
                                        }
                                    }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float s = __uint_as_float(__shfl_sync(0xffffffffu, scale[load][2 * r + h], from));
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                float lo = sum[r][t][2 * h], hi = sum[r][t][2 * h + 1];
                                if constexpr (PIECES > 1) lo += small[r][t][2 * h], hi += small[r][t][2 * h + 1];
                                acc[r][t][h] = fma2(both(lo, hi), both(s, s), acc[r][t][h]);
                            }
                        }
                }
            }
            slot = slot == at0 + (STAGES - 1) * S::SLOT ? at0 : slot + S::SLOT;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' and the cluster's sums ----
    __syncthreads();                                                    // the queues are free
    float *sums = reinterpret_cast<float *>(queue);                     // [warp][8 NT rows of x][16 R weight rows]
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float *to = sums + warp * S::SUMS + (8 * t + 2 * j) * (16 * R) + 16 * r + row + 8 * h;
                asm("mov.b64 {%0, %1}, %2;" : "=f"(to[0]), "=f"(to[16 * R]) : "l"(acc[r][t][h]));
            }
    __syncthreads();
    constexpr int ADD = ALONG_K ? WARPS : 1, TILES = WARPS / ADD;       // warps that share a tile, tiles of the CTA
    if (ALONG_K && parts > 1) {
        for (int i = threadIdx.x; i < S::SUMS; i += THREADS) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < ADD; ++w) sum += sums[w * S::SUMS + i];
            sums[i] = sum;                                              // read by this thread alone before
        }
    }
    if (parts > 1) cluster.sync();
    // CTA `part` stores its share of the outputs
    const int outputs = TILES * x_rows * (16 * R), share = (outputs + parts - 1) / parts;
    for (int i = part * share + threadIdx.x; i < min((part + 1) * share, outputs); i += THREADS) {
        const uint32_t n = i % (16 * R), y = i / (16 * R), m = y % (uint32_t)x_rows, w = y / (uint32_t)x_rows;
        const int64_t first_row = ((int64_t)(blockIdx.x / parts) * TILES + w) * (16 * R);
        if (first_row >= p.outer) continue;
        const int64_t at = min(first_row, max(p.outer - 16 * R, (int64_t)0)) + n;
        if (at >= p.outer) continue;
        float sum = 0.0f;
        float *from = sums + w * S::SUMS + m * (16 * R) + n;
        if (parts > 1) {
            for (int c = 0; c < parts; ++c) sum += *cluster.map_shared_rank(from, c);
        } else {
#pragma unroll
            for (int x = 0; x < ADD; ++x) sum += from[x * S::SUMS];
        }
        sum *= Zero<T>::UP;
        if (p.bias) sum += to_float(reinterpret_cast<const T *>(p.bias)[at]);
        reinterpret_cast<T *>(p.y)[(m0 + m) * p.sy + at] = from_float<T>(sum);
    }
    if (parts > 1) cluster.sync();                                      // shared memory stays until the others have read it
}

// How a call is cut (made of the sizes alone, so that the workspace's size is known before).
struct Plan {
    bool along_k;
    int parts;
    size_t laid;                            // bytes of x laid out in the workspace, 0: in every CTA
};

template <typename T, int NT, int R, int GROUPS, bool ALONG_K, bool BYTES> int launch(MatvecParams p, const Plan &plan, cudaStream_t s) {
    using S = Shape<T, NT, R, GROUPS>;
    const int64_t x_rows = p.rows < 8 * NT ? p.rows : 8 * NT;
    const int all_steps = (int)cdiv(p.inner, 2 * BLOCK);
    p.span = (int32_t)cdiv(all_steps, plan.parts);
    // x whole, or as many of its steps as leave room for a second CTA
    const int64_t phases = cdiv(p.span, (113 * 1024 - S::smem(x_rows, 0)) / (x_rows * S::STEP_BYTES));
    p.phase = phases > 0 ? (int32_t)cdiv(p.span, phases) : 1;
    static bool known[64];
    int dev = 0, launches = 1;
    PITON_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !known[dev]) {
        PITON_CUDA(cudaFuncSetAttribute(matvec_w4_kernel<T, NT, R, GROUPS, ALONG_K, BYTES>, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024));
        if (dev >= 0 && dev < 64) known[dev] = true;
    }
    const dim3 grid((unsigned)(cdiv(p.outer, ALONG_K ? 16 * R : 16 * R * WARPS) * plan.parts), (unsigned)cdiv(p.rows, 8 * NT));
    if (plan.laid) {
        const dim3 laying((unsigned)cdiv(all_steps, 8), (unsigned)p.rows);
        matvec_w4_layout_kernel<T, S::WORDS><<<laying, THREADS, 0, s>>>(p, all_steps);
        launches = 2;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)S::smem(x_rows, p.phase);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)plan.parts;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = plan.laid ? 2 : 1;
    PITON_CUDA(cudaLaunchKernelEx(&cfg, matvec_w4_kernel<T, NT, R, GROUPS, ALONG_K, BYTES>, p));
    return check_launch("matvec_w4", launches);
}

template <typename T, int NT, int R, int GROUPS, bool ALONG_K> int launch(const MatvecParams &p, const Plan &plan, cudaStream_t s) {
    return p.codes_align == 1 ? launch<T, NT, R, GROUPS, ALONG_K, true>(p, plan, s) : launch<T, NT, R, GROUPS, ALONG_K, false>(p, plan, s);
}

template <typename T, int NT, int R, bool ALONG_K> int launch(const MatvecParams &p, const Plan &plan, cudaStream_t s) {
    return p.group_log2 == 7 ? launch<T, NT, R, 1, ALONG_K>(p, plan, s)
           : p.group_log2 == 6 ? launch<T, NT, R, 2, ALONG_K>(p, plan, s) : launch<T, NT, R, 4, ALONG_K>(p, plan, s);
}

template <typename T, int NT> int launch(const MatvecParams &p, const Plan &plan, cudaStream_t s) {
    return plan.along_k ? launch<T, NT, 1, true>(p, plan, s) : launch<T, NT, 2, false>(p, plan, s);
}

Plan plan_of(const piton_matvec_w4_args *a) {
    Plan plan = {true, 1, 0};
    const bool fp32 = a->type == PITON_B200_TYPE_F32;
    const int64_t together = fp32 ? 8 : 16, row_groups = cdiv(a->rows, together);   // rows of x that a CTA takes, CTAs over them
    const int64_t tiles = cdiv(a->outer, 16), sms = num_sms(), steps = cdiv(a->inner, 2 * BLOCK);
    const int64_t most = steps < MAX_PARTS ? steps : MAX_PARTS;
    int64_t parts = 1;                      // a power of two: clusters of 7 took longer than of 4
    // Warps along the rows from 2 x 148 tiles of 16 weight rows on (for every group of rows of x), in as many parts of the inner
    // dimension as two CTAs an SM take in one wave for one such group (28000 x 8192, bf16, one row: 2 parts 37.8 us, 1 part 39.7, 4 parts
    // 41.5; warps along the inner dimension 43.8; fp32, two groups: 2 parts 112, 1 part 135); below that along the inner dimension (4096 x 4096, bf16: 6.0 us, along the rows 8.1; 16 rows of
    // fp32, two groups: 20.4 and 13.7), split further only while SMs are idle and every warp keeps two steps (1024 x 8192: 4
    // parts 5.7 us, 2 parts 6.1).
    if (tiles * row_groups >= 2 * sms && a->outer >= 32) {     // (a warp's 32 weight rows have to exist)
        plan.along_k = false;
        const int64_t groups = cdiv(tiles, 2 * WARPS);
        while (2 * parts <= most && groups * 2 * parts <= 2 * sms) parts *= 2;
    } else {
        while (2 * parts <= most && tiles * 2 * parts <= 2 * sms && steps >= WARPS * 2 * parts) parts *= 2;
    }
    plan.parts = (int)parts;
    // More than 8192 elements of x a CTA are laid out once, in the workspace, by a kernel of their own (bf16, 16 rows by 4096 x 4096: 9.9 us,
    // in every CTA 11.8; fewer do not repay its launch), and more than 2048 of fp32, whose split into pieces is ten times the work.
    const int64_t x_rows = a->rows < together ? a->rows : together;
    if (x_rows * cdiv(steps, parts) * 2 * BLOCK > (fp32 ? 2048 : 8192)) plan.laid = (size_t)(a->rows * steps) * (fp32 ? 1536 : 512);
    return plan;
}

int check_matvec(const piton_matvec_w4_args *a) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->scale_type >= PITON_B200_TYPE_F32 && a->scale_type <= PITON_B200_TYPE_BF16, "unknown scale type %d",
                  a->scale_type);
    PITON_REQUIRE(a->rows >= 0 && a->inner >= 0 && a->outer >= 0, "bad shape");
    PITON_REQUIRE(a->rows <= 65535 && a->outer < (1ll << 31) && a->inner <= (1ll << 30), "rows, inner or outer too large");
    if (a->group != 32 && a->group != 64 && a->group != 128)
        return set_error(PITON_B200_ENOTSUP, "group %d (32, 64, 128)", a->group);
    return PITON_B200_OK;
}

}  // namespace
}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

extern "C" size_t piton_b200_matvec_w4_workspace_size(const piton_matvec_w4_args *a) {
    if (check_matvec(a) != PITON_B200_OK || a->rows == 0 || a->outer == 0) return 0;
    return plan_of(a).laid;
}

extern "C" int piton_b200_matvec_w4(const piton_matvec_w4_args *a, void *stream) {
    if (int rc = check_matvec(a)) return rc;
    if (a->rows == 0 || a->outer == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->y && (a->inner == 0 || (a->x && a->codes && a->scales)), "NULL pointer");
    const Plan plan = plan_of(a);
    if (plan.laid && (!a->workspace || a->workspace_bytes < plan.laid))
        return set_error(PITON_B200_EWORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)a->workspace_bytes,
                         (unsigned long long)plan.laid);
    PITON_REQUIRE(a->workspace % 16 == 0 || !plan.laid, "workspace is not 16-byte aligned");
    MatvecParams p;
    p.laid = plan.laid ? reinterpret_cast<uint8_t *>(a->workspace) : nullptr;
    p.x = reinterpret_cast<const void *>(a->x);
    p.codes = reinterpret_cast<const uint8_t *>(a->codes);
    p.scales = reinterpret_cast<const void *>(a->scales);
    p.zeros = reinterpret_cast<const uint8_t *>(a->zeros);
    p.bias = reinterpret_cast<const void *>(a->bias);
    p.y = reinterpret_cast<void *>(a->y);
    p.rows = a->rows; p.inner = (int32_t)a->inner; p.outer = a->outer;
    p.sx = a->stride_x; p.sc = a->stride_codes; p.ss = a->stride_scales; p.sz = a->stride_zeros; p.sy = a->stride_y;
    p.group_log2 = a->group == 32 ? 5 : a->group == 64 ? 6 : 7; p.scale_type = a->scale_type;
    const uint64_t where = a->codes | (a->outer == 1 ? 0 : (uint64_t)a->stride_codes);   // the rows' alignment
    p.codes_align = where % 16 == 0 ? 16 : where % 4 == 0 ? 4 : 1;
    p.x_aligned = a->x % 16 == 0 && (a->rows == 1 || a->stride_x * (a->type == PITON_B200_TYPE_F32 ? 4 : 2) % 16 == 0);
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        cudaStream_t s = as_stream(stream);
        if constexpr (sizeof(T) == 4) return launch<T, 1>(p, plan, s);  // (three pieces of 16 rows would leave no room for steps)
        else return a->rows <= 8 ? launch<T, 1>(p, plan, s) : launch<T, 2>(p, plan, s);
    });
}
