// y = x W^T (+ bias) with 4-bit weights W[n, k] = scale[n, k / group] (code[n, k] - zero[n, k / group]), for a few rows x.
//
// The codes are read once (N K / 2 bytes) and bound the product up to about 16 rows, so everything is
// arranged around streaming them with few instructions a byte.  A warp takes 16 R weight rows in steps of 256 inner
// elements (128 bytes of a row), copied with cp.async into a queue of its own, so no warp waits for another while it
// streams.  The sums over a group are taken exactly in integers: a nibble is a byte after one mask, and the rows of x
// are laid out as fixed-point numbers of the largest magnitude in their block of 128, two signed 8-bit digits for
// 16-bit types (half a step is 2^-16 of that magnitude; the types' own half steps are larger from 2^-5 of it on for fp16, from
// 2^-8 for bf16) and three for fp32 (2^-24).  x is laid out by a small kernel into a
// workspace, from where a CTA copies its share into shared memory, or by every CTA itself where that share is small.  Codes are the 16-row side of the integer mma.m16n8k32
// and the digits of x its 8-column side; what the accumulators hold is less than 2^22, so started at the bits of
// 1.5 2^23 they are read back as floats by one subtraction.  The zero point's share, zero * sum(x), and the group's
// scale are applied in fp32, two outputs an instruction.  Against products with fp16 or bf16 weights (built first) this takes 3 instead of 9 or 11
// instructions per 8 codes, and instruction issue is what bounds the kernel.  A block of x with a non-finite element
// makes its row of y NaN.
//
// A matrix with many rows gives every warp rows of its own (warps along the rows); one with few splits each
// CTA's inner dimension over its eight warps (warps along the inner dimension).  Either way a cluster of CTAs
// may split the inner dimension further, and adds its parts through distributed shared memory in a fixed order.
//
// Measured: 28000 x 8192, bf16, groups of 128: 1 row 28.0 us (4.2 TB/s), 8 rows 32, groups of 32 with zero points 69;
// 4096 x 4096, bf16: 1 row 5.6 us, 16 rows 9.4; 32768 x 8192, bf16, 16 rows 59 us (2.4 TB/s). Rows of codes on 4 bytes: 8192 x 8200, 1 row
// 15.4 us; on any byte: 4096 x 4098 8.2 us, 28000 x 8194 60 us, copies of 4 bytes a lane where whole rows take 16. A call has 4 to 5 us that do
// not depend on the matrix (launches, x, the cluster's sums); the rest waits for its own chain of loads, integer products
// and fp32 sums with 16 warps an SM: instructions issue in 43 % of the cycles at 16 rows, DRAM is at 27 to 63 %.
// A second buffer of x, filled while the first is used, was slower for 16 rows (62 us).
#include <cooperative_groups.h>

#include <type_traits>

#include "decode.cuh"

namespace piton {
namespace decode {
namespace {

namespace cg = cooperative_groups;

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int BLOCK = 128;                  // inner elements that share a scale of x
constexpr int LINE = 128;                   // bytes of a weight row in a step: two blocks
constexpr int MAX_PARTS = 8;

struct MatvecParams {
    const void *x, *scales, *bias;
    const uint8_t *codes, *zeros;
    void *y;
    int64_t rows, outer, sx, sc, ss, sz, sy;
    int32_t inner, group_log2, scale_type, codes_align, x_aligned;
    uint8_t *digits;                        // x laid out in the workspace, or null: every CTA lays out what it needs
    int32_t span, phase;                    // steps of a CTA's part, and of what shared memory holds of x at a time
};

// An integer v below 2^22 in magnitude, kept as MAGIC + v, read as a float is 1.5 2^23 + v.
constexpr int32_t MAGIC = 0x4B400000;
__device__ __forceinline__ float value_of(int32_t v) { return __int_as_float(v) - 12582912.0f; }

// d = a b + d, or a b + MAGIC.
template <bool FIRST> __device__ __forceinline__ void mma(int32_t (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (FIRST)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(MAGIC));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// The larger magnitude; NaN if one is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
    return d;
}
// Byte `i` of four words.
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int i) {
    const uint32_t two = 0x40 + 0x11 * i;                               // byte i of the first, then of the second
    return __byte_perm(__byte_perm(a, b, two), __byte_perm(c, d, two), 0x5410);
}
__device__ __forceinline__ uint4 load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <int WORDS> __device__ __forceinline__ void load_words(uint32_t (&w)[WORDS], uint32_t at) {
    if constexpr (WORDS == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (WORDS == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

// Two floats in one 64-bit register, and the instructions that take two at a time: half as many to issue.
typedef unsigned long long pair;
__device__ __forceinline__ pair both(float a, float b) {
    pair d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ pair add2(pair a, pair b) {
    pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ pair mul2(pair a, pair b) {
    pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ pair fma2(pair a, pair b, pair c) {
    pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Two sums that were started at MAGIC.
__device__ __forceinline__ pair values_of(int32_t a, int32_t b) {
    return add2(both(__int_as_float(a), __int_as_float(b)), both(-12582912.0f, -12582912.0f));
}

// NT tiles of 8 rows of x, R tiles of 16 weight rows a warp, GROUPS = 128 / group scales of a weight row in a block.
template <typename T, int NT, int R, int GROUPS> struct Shape {
    // Of each group's 32 WORDS elements in a block lane j takes the 8 WORDS from 8 WORDS j on: WORDS words of codes.
    static constexpr int WORDS = 4 / GROUPS;
    // Two stages of 32 weight rows (three: 28000 x 8192 30.0 us, two 28.6 at the time); of 16, three with one tile of x and two with two, whose x
    // takes the room (4096 x 4096, fp32: 8 rows with 4 / 3 / 2 stages 9.7 / 7.9 / 8.1 us, 16 rows with 4 / 2 18.1 / 13.1)
    static constexpr int SLOT = 16 * R * LINE + 128, STAGES = R == 1 && NT == 1 ? 3 : 2, QUEUES = WARPS * STAGES * SLOT;
    static constexpr int DIGITS = sizeof(T) == 4 ? 3 : 2;               // of x; the first holds the most
    static constexpr int SUMS = 8 * NT * 16 * R;                        // outputs of a warp's tile
    // x in shared memory, per row: 16 bytes for every 8 elements (their first two digits), 8 more for fp32 (the third), and per
    // block a scale and each group's sum; paddings put rows that are read together into different banks
    static constexpr int META = 2 * GROUPS;                             // words of a block: 1 + GROUPS, in whole loads
    __host__ __device__ static constexpr int pitch(int steps) { return steps * 512 + 64; }
    __host__ __device__ static constexpr int pitch3(int steps) { return DIGITS == 3 ? steps * 256 + 32 : 0; }
    // shared memory: queues (in the end the warps' sums), x
    static_assert(WARPS * SUMS * 4 <= QUEUES, "the sums fit");
    static int64_t smem(int64_t rows, int64_t steps) {
        return QUEUES + rows * (steps * (512 + (DIGITS == 3 ? 256 : 0)) + 96) + (rows + 1) / 2 * steps * (16 * META);
    }
};

// Where x is laid out: rows of 512 bytes a step (two blocks) of the first two digits, of 256 of the third (fp32), and of META
// words a block.
struct Layout {
    uint8_t *x, *x3;
    float *meta;
    int64_t pitch, pitch3, meta_pitch;
};
// Where the workspace holds all steps of all rows.
template <typename S> __host__ __device__ Layout whole_layout(uint8_t *at, int64_t rows, int64_t steps) {
    Layout l;
    l.pitch = steps * 512, l.pitch3 = S::DIGITS == 3 ? steps * 256 : 0, l.meta_pitch = steps * 4 * S::META;
    l.x = at, l.x3 = at + rows * l.pitch, l.meta = reinterpret_cast<float *>(l.x3 + rows * l.pitch3);
    return l;
}

// Lays out `steps` steps from step0 on of the rows m0 ...: per row and block 16 units of 8 elements, unit 4 c + j for word c of lane
// j (word w of group q: c = q WORDS + w), which faces elements 32 WORDS q + 8 WORDS j + 8 w ... of the block. A unit's bytes are
// its elements 0, 2, 4, 6 (the low nibbles of the word) and 1, 3, 5, 7.
template <typename T, typename S>
__device__ __forceinline__ void lay_out(const MatvecParams &p, int64_t m0, int x_rows, int step0, int steps, const Layout &to) {
    constexpr int WORDS = S::WORDS, DIGITS = S::DIGITS;
    const int count = 2 * steps, units = x_rows * count * 16;
            for (int u0 = 0; u0 < units; u0 += THREADS) {
                const int u = u0 + threadIdx.x, unit = u & 15, c = unit >> 2, b = (u >> 4) % count, m = (u >> 4) / count;
                const int k = (2 * step0 + b) * BLOCK + c / WORDS * (32 * WORDS) + 8 * WORDS * (unit & 3) + 8 * (c % WORDS);
                const bool in = u < units;
                const T *src = reinterpret_cast<const T *>(p.x) + (m0 + (in ? m : 0)) * p.sx + k;
                T v[8];
                if (in && k + 8 <= p.inner && p.x_aligned) {
    #pragma unroll
                    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(src)[i];
                } else {
    #pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = in && k + i < p.inner ? src[i] : from_float<T>(0.0f);
                }
                float f[8], top = 0.0f;
    #pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = to_float(v[i]), top = max_abs(top, f[i]);
    #pragma unroll
                for (int o = 1; o < 16; o <<= 1) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, o));
                // the largest magnitude becomes 127 in the first digit and 0 in the others
                constexpr float LIMIT = DIGITS == 3 ? 127.0f * 65536.0f : 127.0f * 256.0f;
                const bool finite = top < INFINITY;
                const float up = !finite ? 0.0f : fminf(LIMIT / fmaxf(top, 1e-37f), 8.5070592e37f), down = !finite ? __int_as_float(0x7FC00000) : 1.0f / up;
                // with 128 added to every digit but the first the digits are the bytes of the sum, those less 128 of them signed
                uint32_t t[8], digit[3][2] = {};
    #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (DIGITS == 3) t[i] = (uint32_t)(finite ? __float2int_rn(f[i] * up) + 0x8080 : 0x8080);
                    else t[i] = finite ? __float_as_uint(fmaf(f[i], up, 12582912.0f + 128.0f)) : 0x80u;
                }
                int32_t sum = 0;
    #pragma unroll
                for (int d = 0; d < DIGITS; ++d) {
                    int32_t own = 0;
    #pragma unroll
                    for (int h = 0; h < 2; ++h) {                           // elements 0, 2, 4, 6 and 1, 3, 5, 7
                        digit[d][h] = bytes_of(t[h], t[2 + h], t[4 + h], t[6 + h], DIGITS - 1 - d) ^ (d ? 0x80808080u : 0u);
                        own = __dp4a((int)digit[d][h], 0x01010101, own);
                    }
                    sum = 256 * sum + own;
                }
    #pragma unroll
                for (int o = 1; o < 4 * WORDS; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);    // a group's units: below 2^30
                if (in) {
                    *reinterpret_cast<uint4 *>(to.x + m * to.pitch + (b * 16 + unit) * 16) = make_uint4(digit[0][0], digit[0][1], digit[1][0], digit[1][1]);
                    if constexpr (DIGITS == 3) *reinterpret_cast<uint2 *>(to.x3 + m * to.pitch3 + (b * 16 + unit) * 8) = make_uint2(digit[2][0], digit[2][1]);
                    float *about = to.meta + (m >> 1) * to.meta_pitch + b * (2 * S::META) + ((m0 + m) & 1);
                    if (unit == 0) about[0] = down;
                    if (unit % (4 * WORDS) == 0) about[2 + 2 * (unit / (4 * WORDS))] = (float)sum;
                }
            }
}

// x laid out once for all CTAs, which would otherwise repeat it for every 256 weight rows: a thread a unit.
template <typename T, typename S> __global__ void __launch_bounds__(THREADS) matvec_w4_digits_kernel(const MatvecParams p, int all_steps, bool early) {
    if (early) asm volatile("griddepcontrol.launch_dependents;");   // the product may start on its weights, and waits before it reads x
    const int step = blockIdx.x * 8, m = blockIdx.y;
    Layout to = whole_layout<S>(p.digits, p.rows, all_steps);
    to.x += m * to.pitch + step * 512, to.x3 += m * to.pitch3 + step * 256, to.meta += (m >> 1) * to.meta_pitch + step * 4 * S::META;
    lay_out<T, S>(p, m, 1, step, min(8, all_steps - step), to);
    if (!early) asm volatile("griddepcontrol.launch_dependents;");
}

// ALONG_K: the CTA's warps share 16 R weight rows and split the inner dimension; otherwise each has rows of its own.
template <typename T, int NT, int R, int GROUPS, bool ALONG_K, bool BYTES>
__global__ void __launch_bounds__(THREADS, 2) matvec_w4_kernel(const MatvecParams p) {
    using S = Shape<T, NT, R, GROUPS>;
    constexpr int WORDS = S::WORDS, STAGES = S::STAGES, STRIDE = ALONG_K ? WARPS : 1, DIGITS = S::DIGITS, STEP = 2 * BLOCK;
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
                    if (R > 1 || 4 * i + (lane >> 3) < rows) copy16(dst[i & 1] + 512 * i, src);
                    src += 4 * p.sc;
                }
            } else if (whole && p.codes_align == 4) {                   // a row a copy
                const uint8_t *src = codes + 4 * lane;
#pragma unroll 8
                for (int r = 0; r < 16 * R; ++r) {
                    if (R > 1 || r < rows) copy4(fill + 128 * r + ((lane >> 2) ^ (r & 7)) * 16 + 4 * (lane & 3), src);
                    src += p.sc;
                }
            } else {                                                    // the last step, or rows that are not aligned: words that hold a byte of the row
                const uint8_t *src = codes;
                const int64_t left = (p.inner + 1) / 2 - (int64_t)(step0 + own0 + issued * STRIDE) * LINE;
#pragma unroll 4
                for (int r = 0; r < rows; ++r) {
                    const int before = (int)(reinterpret_cast<uintptr_t>(src) & 3);
                    if (4 * lane - before < left) copy4(fill + 128 * r + ((lane >> 2) ^ (r & 7)) * 16 + 4 * (lane & 3), src - before + 4 * lane);
                    src += p.sc;
                }
                src = codes + lane * p.sc;
                const int before = (int)(reinterpret_cast<uintptr_t>(src) & 3);
                if (before && lane < rows && LINE - before < left) copy4(fill + 16 * R * LINE + 4 * lane, src - before + LINE);
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

    // ---- x in shared memory ----
    uint8_t *xs = queue + S::QUEUES;
    uint8_t *x3 = xs + x_rows * S::pitch(p.phase);
    float *meta = reinterpret_cast<float *>(x3 + x_rows * S::pitch3(p.phase));      // [x row][block of the phase][META]
    // rows of x past the last read the last: a column of the product depends on its own row alone
    uint32_t x_at[NT], x3_at[NT];
    uint32_t meta_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int m = min(8 * t + g, x_rows - 1);
        x_at[t] = (uint32_t)__cvta_generic_to_shared(xs) + m * S::pitch(p.phase) + 16 * j;
        x3_at[t] = (uint32_t)__cvta_generic_to_shared(x3) + m * S::pitch3(p.phase) + 8 * j;
        meta_at[t] = (uint32_t)__cvta_generic_to_shared(meta + min(4 * t + j, (x_rows - 1) >> 1) * (4 * p.phase * S::META));
    }

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
        if (p.digits) {                                                 // 16 bytes at a time, as they lie in the workspace
            const Layout from = whole_layout<S>(p.digits, p.rows, (p.inner + STEP - 1) / STEP);
            if (phase0 == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
            auto copy = [&](uint8_t *to, int to_pitch, const uint8_t *src, int64_t src_pitch, int row_bytes, int rows_of) {
                for (int m = warp; m < rows_of; m += WARPS)
#pragma unroll 4
                    for (int i = 16 * lane; i < row_bytes; i += 512) copy16((uint32_t)__cvta_generic_to_shared(to + m * to_pitch + i), src + m * src_pitch + i);
            };
            const int64_t at = step0 + phase0;
            copy(xs, S::pitch(p.phase), from.x + m0 * from.pitch + at * 512, from.pitch, count * 512, x_rows);
            if constexpr (DIGITS == 3) copy(x3, S::pitch3(p.phase), from.x3 + m0 * from.pitch3 + at * 256, from.pitch3, count * 256, x_rows);
            copy(reinterpret_cast<uint8_t *>(meta), 16 * S::META * p.phase,
                 reinterpret_cast<const uint8_t *>(from.meta + m0 / 2 * from.meta_pitch + at * 4 * S::META), 4 * from.meta_pitch, count * 16 * S::META,
                 (x_rows + 1) / 2);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        } else {
            lay_out<T, S>(p, m0, x_rows, step0 + phase0, count, {xs, x3, meta, S::pitch(p.phase), S::pitch3(p.phase), 4 * p.phase * S::META});
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
                pair about[NT][S::META];                                // the block's scales, then its groups' sums
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i <= GROUPS; i += 2) {
                        const uint32_t from = meta_at[t] + (b0 + b) * (8 * S::META) + 8 * i;
                        if (i < GROUPS) asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(about[t][i]), "=l"(about[t][i + 1]) : "r"(from) : "memory");
                        else asm volatile("ld.shared.u64 %0, [%1];" : "=l"(about[t][i]) : "r"(from) : "memory");
                    }
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) {
                    uint4 x12[NT][WORDS];
                    uint2 x3v[NT][WORDS];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < WORDS; ++i) {
                            x12[t][i] = load16(x_at[t] + (b0 + b) * 256 + (q * WORDS + i) * 64);
                            x3v[t][i] = make_uint2(0, 0);
                            if constexpr (DIGITS == 3)
                                asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x3v[t][i].x), "=r"(x3v[t][i].y)
                                             : "r"(x3_at[t] + (b0 + b) * 128 + (q * WORDS + i) * 32) : "memory");
                        }
                    }
                    constexpr int LAST = LOADS - 1;
                    const int load = GROUPS == 4 ? b & LAST : 0;
                    const int from = (lane & ~3) | (GROUPS == 1 ? (turn & 1) * 2 + b : GROUPS == 2 ? 2 * b + q : q);
                    const uint32_t z = __shfl_sync(0xffffffffu, zeros[load], from);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        pair s2[2], z2[2];                              // scales and zero points, the latter negative
                        uint32_t w[2][WORDS];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float s = __uint_as_float(__shfl_sync(0xffffffffu, scale[load][2 * r + h], from));
                            const float minus = -value_of(MAGIC | (z >> (16 * r + 8 * h) & 255));
                            s2[h] = both(s, s), z2[h] = both(minus, minus);
                            // WORDS words of codes from byte 64 b + 16 WORDS q + 4 WORDS j of row 16 r + row + 8 h
                            load_words(w[h], (wat ^ (64 * b + 16 * WORDS * q)) + (16 * r + 8 * h) * LINE);
                            if constexpr (BYTES) {
                                const int next = 16 * b + 4 * WORDS * q + WORDS * j + WORDS;    // the word after them
                                uint32_t v[1];
                                load_words(v, next == LINE / 4 ? slot + 16 * R * LINE + 4 * (16 * r + row + 8 * h)
                                                               : slot + (16 * r + row + 8 * h) * LINE + ((next >> 2) ^ (row & 7)) * 16 + 4 * (next & 3));
#pragma unroll
                                for (int i = 0; i < WORDS; ++i) w[h][i] = __funnelshift_r(w[h][i], i + 1 < WORDS ? w[h][i + 1] : v[0], before >> (8 * (2 * r + h)));
                            }
                        }
                        int32_t sum[NT][DIGITS][4];
#pragma unroll
                        for (int i = 0; i < WORDS; ++i) {
                            constexpr uint32_t LOW = 0x0F0F0F0Fu;
                            const uint32_t a[4] = {w[0][i] & LOW, w[1][i] & LOW, w[0][i] >> 4 & LOW, w[1][i] >> 4 & LOW};
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                const uint32_t x[6] = {x12[t][i].x, x12[t][i].y, x12[t][i].z, x12[t][i].w, x3v[t][i].x, x3v[t][i].y};
#pragma unroll
                                for (int d = 0; d < DIGITS; ++d) {
                                    if (i == 0) mma<true>(sum[t][d], a, x[2 * d], x[2 * d + 1]);
                                    else mma<false>(sum[t][d], a, x[2 * d], x[2 * d + 1]);
                                }
                            }
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                pair v = values_of(sum[t][0][2 * h], sum[t][0][2 * h + 1]);
#pragma unroll
                                for (int d = 1; d < DIGITS; ++d) v = fma2(v, both(256.0f, 256.0f), values_of(sum[t][d][2 * h], sum[t][d][2 * h + 1]));
                                v = fma2(z2[h], about[t][1 + q], v);
                                acc[r][t][h] = fma2(v, mul2(about[t][0], s2[h]), acc[r][t][h]);
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
        if (p.bias) sum += to_float(reinterpret_cast<const T *>(p.bias)[at]);
        reinterpret_cast<T *>(p.y)[(m0 + m) * p.sy + at] = from_float<T>(sum);
    }
    if (parts > 1) cluster.sync();                                      // shared memory stays until the others have read it
}

// How a call is cut (made of the sizes alone, so that the workspace's size is known before).
struct Plan {
    bool along_k;
    int parts;
    size_t digits;                          // bytes of x laid out in the workspace, 0: in every CTA
};

template <typename T, int NT, int R, int GROUPS, bool ALONG_K, bool BYTES> int launch(MatvecParams p, const Plan &plan, cudaStream_t s) {
    using S = Shape<T, NT, R, GROUPS>;
    const int64_t x_rows = p.rows < 8 * NT ? p.rows : 8 * NT;
    const int all_steps = (int)cdiv(p.inner, 2 * BLOCK);
    p.span = (int32_t)cdiv(all_steps, plan.parts);
    // x whole, or as many of its steps as leave room for a second CTA
    p.phase = p.span > 0 ? p.span : 1;
    while (S::smem(x_rows, p.phase) > 113 * 1024 && p.phase > 1) p.phase = (p.phase + 1) / 2;
    static bool known[64];
    int dev = 0, launches = 1;
    PITON_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !known[dev]) {
        PITON_CUDA(cudaFuncSetAttribute(matvec_w4_kernel<T, NT, R, GROUPS, ALONG_K, BYTES>, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024));
        if (dev >= 0 && dev < 64) known[dev] = true;
    }
    const dim3 grid((unsigned)(cdiv(p.outer, ALONG_K ? 16 * R : 16 * R * WARPS) * plan.parts), (unsigned)cdiv(p.rows, 8 * NT));
    if (plan.digits) {
        const dim3 laying((unsigned)cdiv(all_steps, 8), (unsigned)p.rows);
        // The product starts while x is laid out, unless its clusters would then not all find room at once: 4096 x 4096, one
        // row, 256 + 2 CTAs: 5.8 us, after it 6.4; 8192 x 8192, 5 rows, bf16, 32 clusters + 20 CTAs: 17.5 us, after it 12.9.
        const bool early = plan.parts == 1 || (int64_t)grid.x * grid.y + (int64_t)laying.x * laying.y <= 272;
        matvec_w4_digits_kernel<T, S><<<laying, THREADS, 0, s>>>(p, all_steps, early);
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
    cfg.numAttrs = plan.digits ? 2 : 1;
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
    const int64_t tiles = cdiv(a->outer, 16), sms = num_sms(), steps = cdiv(a->inner, 2 * BLOCK);
    const int64_t most = steps < MAX_PARTS ? steps : MAX_PARTS;
    int64_t parts = 1;                      // a power of two: clusters of 7 took longer than of 4
    // Warps along the rows from 2 x 148 tiles of 16 weight rows on, in as many parts of the inner dimension as two CTAs an SM
    // take in one wave (28000 x 8192, bf16, one row: 2 parts 29.4 us, 1 part 36.6, 4 parts 32.2; warps along the inner
    // dimension 40); below that along the inner dimension (4096 x 4096: 6.2 us, along the rows 6.2 to 9), split
    // further only while SMs are idle and every warp keeps two steps (1024 x 8192: 4 parts 5.5 us, 1 part 7.8).
    if (tiles >= 2 * sms) {
        plan.along_k = false;
        const int64_t groups = cdiv(tiles, 2 * WARPS);
        while (2 * parts <= most && groups * 2 * parts <= 2 * sms) parts *= 2;
    } else {
        while (2 * parts <= most && tiles * 2 * parts <= 2 * sms && steps >= WARPS * 2 * parts) parts *= 2;
    }
    plan.parts = (int)parts;
    // More than 2048 elements of x a CTA are laid out once in the workspace, by a kernel of their own (bf16, 8192 elements, 4 rows
    // by 2048 x 2048: 4.6 us, in every CTA 6.0; 2048 elements, 8 rows by 8192 x 2048: 7.1 and 6.7; 65536 elements, 16 rows by
    // 4096 x 4096: 9.3 and 28).
    const int64_t x_rows = a->rows < 16 ? a->rows : 16;
    if (x_rows * cdiv(steps, parts) * 2 * BLOCK > 2048) {
        const int64_t fp32 = a->type == PITON_B200_TYPE_F32;
        plan.digits = (size_t)(a->rows * steps) * (512 + (fp32 ? 256 : 0)) + (size_t)((a->rows + 1) / 2 * steps) * (32 * (128 / a->group));
    }
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
    return plan_of(a).digits;
}

extern "C" int piton_b200_matvec_w4(const piton_matvec_w4_args *a, void *stream) {
    if (int rc = check_matvec(a)) return rc;
    if (a->rows == 0 || a->outer == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->y && (a->inner == 0 || (a->x && a->codes && a->scales)), "NULL pointer");
    const Plan plan = plan_of(a);
    if (plan.digits && (!a->workspace || a->workspace_bytes < plan.digits))
        return set_error(PITON_B200_EWORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)a->workspace_bytes,
                         (unsigned long long)plan.digits);
    PITON_REQUIRE(a->workspace % 16 == 0 || !plan.digits, "workspace is not 16-byte aligned");
    MatvecParams p;
    p.digits = plan.digits ? reinterpret_cast<uint8_t *>(a->workspace) : nullptr;
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
        return a->rows <= 8 ? launch<T, 1>(p, plan, s) : launch<T, 2>(p, plan, s);
    });
}
