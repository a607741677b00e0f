// Appending to a paged 8-bit cache: keys rotated by position, keys and values quantised to e4m3
// with a power-of-two scale per (page, head), queries rotated in the same launch.
//
// A unit is one page that one sequence's new tokens touch; a task is one (unit, head, key or value):
// the block's largest finite magnitude, its scale, the older tokens requantised where the scale
// grows, the new tokens' codes.  The scale is a power of two, so dividing by it is exact and a
// growing scale moves old codes without a second rounding until they reach e4m3's subnormals; the
// format's relative precision does not depend on where in a binade the scale sits.
//
// The bytes in and out bound it.  Every element is read once, 16 bytes at a time: a thread takes a pair of
// 16-byte pieces whose elements rotate with one another, keeps the rotated values in registers until the
// block's scale is known, and reads its rows of the rotation tables once for all heads that it walks.
// Rows that do not lie on 16 bytes, or rotate in pairs of pieces that do not, take the element-by-element kernel.
//
// Measured: long prompts, 742 MB in and out: 152 us (4.9 TB/s); ragged prompts, 304 MB: 59 us (5.2 TB/s); 256 sequences, a token
// each: 6.5 us; one token: 3.4 us. Where the long prompts took 148 us, a launch of its own for the queries took 205, no load of the next
// head while the last is stored 215.
#include "decode.cuh"

namespace piton {
namespace decode {

__device__ int g_append_status = 0;

namespace {

constexpr int THREADS = 128;

struct AppendParams {
    const void *k, *v, *q;
    void *q_out;
    uint8_t *codes[2];
    float *scale[2];
    const int32_t *table, *starts, *cu;
    int32_t *lengths;
    const float *cos_table, *sin_table;
    int64_t batch, tokens, kv_heads, q_heads, page_size, num_pages, table_width, table_stride;
    int64_t st[2], sh[2], sqt, sqh, sot, soh;   // strides of k and v, q, q_out
    int64_t rope_len, units, uniform, unit_blocks;
    int32_t dim, rot, interleaved;
};

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_append_status, 0, code); }

// The least power of two s in [2^-120, 2^120] with a <= 448 s (a >= 0): 448 = 1.75 * 2^8, so the
// exponent is a's less 8, one more when its significand exceeds 1.75.
__device__ __forceinline__ float block_scale(float a) {
    const uint32_t u = __float_as_uint(a);
    int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    if ((u >> 23) == 0) e = 7;                                       // zero and denormals: the least scale
    e = min(max(e, 7), 247);
    return __uint_as_float((uint32_t)e << 23);
}

__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.0f; }

// Element d of the row x rotated by the row (c, s): every product and sum rounded by itself, so the
// result does not depend on how a compiler contracts them.
template <typename T>
__device__ __forceinline__ float rotated(const T *x, int d, const float *c, const float *s, int rot, bool interleaved) {
    const float a = to_float(x[d]);
    if (d >= rot) return a;
    const int half = rot >> 1;
    const bool second = interleaved ? (d & 1) : d >= half;
    const int i = interleaved ? d >> 1 : (second ? d - half : d);
    const float b = to_float(x[interleaved ? d ^ 1 : (second ? d - half : d + half)]);
    return second ? __fadd_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i])) : __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
}

// The sequence of new token t (ragged): the last b with cu[b] <= t.
__device__ __forceinline__ int64_t sequence_of_token(const AppendParams &p, int64_t t) {
    if (!p.cu) return t / p.uniform;
    int64_t lo = 0, hi = p.batch - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Units are numbered sequence by sequence.  Uniform: a fixed number each.  Ragged: sequence b's
// start at cu[b] / page_size + 2 b, which leaves it at least the n / page_size + 2 pages that n
// tokens can touch.
__device__ __forceinline__ int64_t first_unit(const AppendParams &p, int64_t b) {
    return (p.cu ? min(max((int64_t)p.cu[b], (int64_t)0), p.tokens) / p.page_size : 0) + 2 * b;
}

// The sequences' new lengths, a thread each; 0 for one that is refused because it starts below 0, so that none of its keys is attended.
__device__ __forceinline__ void write_lengths(const AppendParams &p) {
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < p.batch; b += (int64_t)gridDim.x * blockDim.x) {
        const int64_t start = p.starts[b];
        if (p.lengths) p.lengths[b] = start < 0 ? 0 : (int32_t)min(start + span_of(p.cu, b, p.uniform, p.tokens).n, (int64_t)INT32_MAX);
        if (start < 0 || (p.cu && (p.cu[b] < 0 || p.cu[b + 1] < p.cu[b] || p.cu[b + 1] > p.tokens))) record_status(STATUS_BAD_POSITION);
    }
}

// Tokens at positions [lo, hi) that the rotation tables have rows for.
__device__ __forceinline__ int live_tokens(const AppendParams &p, int64_t lo, int64_t hi) {
    return (int)((p.rot ? min(max(p.rope_len, lo), hi) : hi) - lo);
}

// Zeros to bytes [from, to) of a page's heads.
__device__ __forceinline__ void clear_codes(const AppendParams &p, int which, int64_t page, int head0, int head1, int from, int to, int worker, int workers) {
    const int64_t bytes = p.page_size * p.dim;
    for (int h = head0; h < head1; ++h)
        for (int i = from + 16 * worker; i < to; i += 16 * workers)
            *reinterpret_cast<uint4 *>(p.codes[which] + (page * p.kv_heads + h) * bytes + i) = uint4();
}

// Whether query token t is rotated: it has to belong to the sequence and to have a position that the tables hold; it is 0 otherwise.
__device__ __forceinline__ bool rotates(const AppendParams &p, const Span &sp, int64_t t, int64_t start, bool report) {
    if (t < sp.t0 || t >= sp.t0 + sp.n) return false;                // a token of no sequence
    if (start >= 0 && (p.rot == 0 || start + t - sp.t0 < p.rope_len)) return true;
    if (report) record_status(STATUS_BAD_POSITION);
    return false;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(const AppendParams p) {
    const int tid = threadIdx.x;
    write_lengths(p);
    if (blockIdx.x >= p.unit_blocks) {                               // queries: a warp per (token, head)
        const int64_t row = ((int64_t)blockIdx.x - p.unit_blocks) * (THREADS / 32) + (tid >> 5);
        if (row >= p.tokens * p.q_heads) return;
        const int64_t t = row / p.q_heads, h = row % p.q_heads, b = sequence_of_token(p, t);
        const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
        const int64_t pos = (int64_t)p.starts[b] + t - sp.t0;
        const T *x = reinterpret_cast<const T *>(p.q) + t * p.sqt + h * p.sqh;
        T *y = reinterpret_cast<T *>(p.q_out) + t * p.sot + h * p.soh;
        if (!rotates(p, sp, t, p.starts[b], (tid & 31) == 0)) {
            for (int d = tid & 31; d < p.dim; d += 32) y[d] = from_float<T>(0.0f);
            return;
        }
        const float *c = p.cos_table + pos * (p.rot >> 1), *s = p.sin_table + pos * (p.rot >> 1);
        for (int d = tid & 31; d < p.dim; d += 32) y[d] = from_float<T>(rotated(x, d, c, s, p.rot, p.interleaved));
        return;
    }
    const int64_t per_unit = 2 * p.kv_heads;
    const int64_t unit = blockIdx.x / per_unit;
    const int64_t h = (blockIdx.x % per_unit) >> 1;
    const int which = blockIdx.x & 1;
    int64_t b, j;
    if (!p.cu) {
        const int64_t each = p.units / p.batch;
        b = unit / each;
        j = unit % each;
    } else {
        int64_t lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (first_unit(p, mid) <= unit) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        j = unit - first_unit(p, b);
    }
    const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
    const int64_t start = p.starts[b], end = start + sp.n;
    if (start < 0) return;                                           // (reported with the lengths)
    const int64_t place = start / p.page_size + j;                   // this unit's page of the sequence
    const int64_t page0 = place * p.page_size;
    const int64_t lo = max(start, page0), hi = min(end, page0 + p.page_size);
    if (lo >= hi) return;
    if (place >= p.table_width) {
        if (tid == 0) record_status(STATUS_BAD_POSITION);
        return;
    }
    const int64_t page = p.table[b * p.table_stride + place];
    if (page < 0 || page >= p.num_pages) {
        if (tid == 0) record_status(STATUS_BAD_PAGE);
        return;
    }
    const int rot = which == 0 ? p.rot : 0;
    const T *x = reinterpret_cast<const T *>(which == 0 ? p.k : p.v) + (sp.t0 + lo - start) * p.st[which] + h * p.sh[which];
    uint8_t *codes = p.codes[which] + (page * p.kv_heads + h) * p.page_size * p.dim;
    float *scale = p.scale[which] + page * p.kv_heads + h;
    const int count = (int)(hi - lo) * p.dim, held = (int)(lo - page0);
    const int live = live_tokens(p, lo, hi);                         // the others have no rotation: zeros
    if (lo + live < hi && tid == 0) record_status(STATUS_BAD_POSITION);
    auto value = [&](int i) {
        const int t = i / p.dim, d = i % p.dim;
        if (t >= live) return 0.0f;
        const int64_t row = (lo + t) * (rot >> 1);
        return rotated(x + t * p.st[which], d, p.cos_table + row, p.sin_table + row, rot, p.interleaved);
    };
    float a = 0.0f;
    for (int i = tid; i < count; i += THREADS) a = fmaxf(a, finite_abs(value(i)));
    __shared__ float red[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((tid & 31) == 0) red[tid >> 5] = a;
    const float before = held ? *scale : 0.0f;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) a = fmaxf(a, red[w]);
    const float s = fmaxf(block_scale(a), before);
    const float inv = 1.0f / s;                                      // a power of two: exact
    if (held && s > before) {
        const float ratio = before * inv;
        for (int i = tid; i < held * p.dim; i += THREADS) codes[i] = float_to_e4m3(e4m3_to_float(codes[i]) * ratio);
    }
    for (int i = tid; i < count; i += THREADS) {
        const float y = value(i);
        codes[held * p.dim + i] = float_to_e4m3(isfinite(y) ? y * inv : __int_as_float(0x7FC00000));
    }
    if (tid == 0) *scale = s;
}


// ---- rows on 16 bytes ----

// V = 16 / sizeof(T) elements a piece; pair u of a head's dim / (2 V): pieces at V u and rot / 2 + V u where they rotate in
// halves, else two neighbouring pieces from 2 V u on (interleaved pairs, or past rot).
template <typename T> struct Pair {
    static constexpr int V = 16 / sizeof(T);
    float a[V], b[V];
};
struct PairPlace {
    int a, b;              // element offsets in the head
    bool turns, inside;    // rotates; with pairs inside a piece
};
template <typename T> __device__ __forceinline__ PairPlace place_of(int u, int rot, bool interleaved) {
    constexpr int V = 16 / sizeof(T);
    const bool turns = 2 * V * u < rot, halves = turns && !interleaved;
    return {halves ? V * u : 2 * V * u, halves ? (rot >> 1) + V * u : 2 * V * u + V, turns, interleaved};
}
__device__ __forceinline__ void unpack(float (&f)[4], const uint4 &r, float) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void unpack(float (&f)[8], const uint4 &r, __half) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = x.x, f[2 * i + 1] = x.y;
    }
}
__device__ __forceinline__ void unpack(float (&f)[8], const uint4 &r, __nv_bfloat16) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ uint4 packed(const float (&f)[4], float) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 packed(const float (&f)[8], __half) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 packed(const float (&f)[8], __nv_bfloat16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The larger magnitude; NaN if one is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
    return d;
}
__device__ __forceinline__ uint4 load_stream(const void *p) { return __ldcs(reinterpret_cast<const uint4 *>(p)); }

// Rotates a pair by its row of the tables (c, s: V values from element V u of the row).
template <typename T> __device__ __forceinline__ void turn(Pair<T> &x, const float (&c)[Pair<T>::V], const float (&s)[Pair<T>::V], const PairPlace &at) {
    constexpr int V = Pair<T>::V;
    if (!at.turns) return;
    if (at.inside) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float a0 = x.a[i], a1 = x.a[i + 1], b0 = x.b[i], b1 = x.b[i + 1];
            x.a[i] = __fsub_rn(__fmul_rn(a0, c[i / 2]), __fmul_rn(a1, s[i / 2]));
            x.a[i + 1] = __fadd_rn(__fmul_rn(a1, c[i / 2]), __fmul_rn(a0, s[i / 2]));
            x.b[i] = __fsub_rn(__fmul_rn(b0, c[(V + i) / 2]), __fmul_rn(b1, s[(V + i) / 2]));
            x.b[i + 1] = __fadd_rn(__fmul_rn(b1, c[(V + i) / 2]), __fmul_rn(b0, s[(V + i) / 2]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float a = x.a[i], b = x.b[i];
            x.a[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
            x.b[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
        }
    }
}
template <int V> __device__ __forceinline__ void load_row(float (&f)[V], const float *p) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const float4 r = __ldg(reinterpret_cast<const float4 *>(p + i));
        f[i] = r.x, f[i + 1] = r.y, f[i + 2] = r.z, f[i + 3] = r.w;
    }
}
template <int V> __device__ __forceinline__ void store_codes(uint8_t *to, const float (&f)[V], float inv, bool all_finite) {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        float2 y = make_float2(f[i] * inv, f[i + 1] * inv);
        if (!all_finite) {
            y.x = isfinite(f[i]) ? y.x : __int_as_float(0x7FC00000);
            y.y = isfinite(f[i + 1]) ? y.y : __int_as_float(0x7FC00000);
        }
        const uint32_t two = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
        if (i % 4 == 0) w[i / 4] = two;
        else w[i / 4] |= two << 16;
    }
    if constexpr (V == 4) *reinterpret_cast<uint32_t *>(to) = w[0];
    else *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
}

constexpr int WIDE = 256;      // threads of a CTA

// A task by TT threads (a warp or the CTA), at most PASSES pairs a thread; the CTA's tasks are `heads_each` heads of one unit,
// one after the other (TT = WIDE) or WIDE / 32 of the list, a warp each.
template <typename T, int D, int TT, int PASSES>
__global__ void __launch_bounds__(WIDE, PASSES == 1 ? 4 : PASSES == 2 ? 3 : PASSES == 4 ? 2 : 1) kv_append_wide_kernel(const AppendParams p, int heads_each, int q_pieces) {
    constexpr int V = 16 / sizeof(T), UPH = D / (2 * V);             // pairs of a head
    const int tid = threadIdx.x, lane = tid & 31;
    write_lengths(p);
    if (blockIdx.x >= p.unit_blocks) {                               // queries: a warp per token and piece of the heads
        const int64_t item = ((int64_t)blockIdx.x - p.unit_blocks) * (WIDE / 32) + (tid >> 5);
        const int64_t t = item / q_pieces;
        if (t >= p.tokens) return;
        const int64_t b = sequence_of_token(p, t);
        const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
        const int64_t pos = (int64_t)p.starts[b] + t - sp.t0;
        const bool named = rotates(p, sp, t, p.starts[b], lane == 0);
        constexpr int SIDE = 32 / UPH;                               // heads at once
        const int u = lane % UPH;
        const PairPlace at = place_of<T>(u, p.rot, p.interleaved);
        float c[V], s[V];
        if (at.turns && named) {
            load_row(c, p.cos_table + pos * (p.rot >> 1) + V * u);
            load_row(s, p.sin_table + pos * (p.rot >> 1) + V * u);
        }
        const T *x = reinterpret_cast<const T *>(p.q) + t * p.sqt;
        T *y = reinterpret_cast<T *>(p.q_out) + t * p.sot;
        const int heads = (int)p.q_heads, step = SIDE * q_pieces;
        int h = (int)(item % q_pieces) * SIDE + lane / UPH;
        if (!named) {
            for (; h < heads; h += step) *reinterpret_cast<uint4 *>(y + h * p.soh + at.a) = *reinterpret_cast<uint4 *>(y + h * p.soh + at.b) = uint4();
            return;
        }
        for (; h < heads; h += 2 * step) {                           // two heads in flight
            const bool more = h + step < heads;
            const T *x0 = x + h * p.sqh, *x1 = x + (int64_t)(h + step) * p.sqh;
            const uint4 a0 = load_stream(x0 + at.a), b0 = load_stream(x0 + at.b);
            uint4 a1 = {}, b1 = {};
            if (more) a1 = load_stream(x1 + at.a), b1 = load_stream(x1 + at.b);
            Pair<T> v;
            unpack(v.a, a0, T());
            unpack(v.b, b0, T());
            turn<T>(v, c, s, at);
            T *y0 = y + h * p.soh, *y1 = y + (int64_t)(h + step) * p.soh;
            *reinterpret_cast<uint4 *>(y0 + at.a) = packed(v.a, T());
            *reinterpret_cast<uint4 *>(y0 + at.b) = packed(v.b, T());
            if (more) {
                unpack(v.a, a1, T());
                unpack(v.b, b1, T());
                turn<T>(v, c, s, at);
                *reinterpret_cast<uint4 *>(y1 + at.a) = packed(v.a, T());
                *reinterpret_cast<uint4 *>(y1 + at.b) = packed(v.b, T());
            }
        }
        return;
    }
    const int worker = tid % TT;
    const int pieces = (int)((p.kv_heads + heads_each - 1) / heads_each);    // of a unit's heads, keys and values apart
    const int64_t task = TT == WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (WIDE / TT) + tid / TT;
    const int64_t unit = task / (2 * pieces);
    if (unit >= p.units) return;
    const int which = (int)(task % (2 * pieces)) & 1, head0 = ((int)(task % (2 * pieces)) >> 1) * heads_each;
    int64_t b, j;
    if (!p.cu) {
        const int64_t each = p.units / p.batch;
        b = unit / each;
        j = unit % each;
    } else {
        int64_t lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (first_unit(p, mid) <= unit) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        j = unit - first_unit(p, b);
    }
    const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
    const int64_t start = p.starts[b], end = start + sp.n;
    if (start < 0) return;                                           // (reported with the lengths)
    const int64_t place = start / p.page_size + j, page0 = place * p.page_size;
    const int64_t lo = max(start, page0), hi = min(end, page0 + p.page_size);
    if (lo >= hi) return;
    if (place >= p.table_width) {
        if (worker == 0) record_status(STATUS_BAD_POSITION);
        return;
    }
    const int64_t page = p.table[b * p.table_stride + place];
    if (page < 0 || page >= p.num_pages) {
        if (worker == 0) record_status(STATUS_BAD_PAGE);
        return;
    }
    const int rot = which == 0 ? p.rot : 0, count = live_tokens(p, lo, hi), held = (int)(lo - page0), u = worker % UPH;
    if (lo + count < hi) {                                           // tokens that have no rotation
        if (worker == 0) record_status(STATUS_BAD_POSITION);
        clear_codes(p, which, page, head0, min(head0 + heads_each, (int)p.kv_heads), (held + count) * D, (int)(hi - page0) * D, worker, TT);
    }
    const PairPlace at = place_of<T>(u, rot, p.interleaved);
    constexpr int TOKENS = TT / UPH;                                 // a pass
    const int token = worker / UPH;
    const int64_t st = p.st[which], sh = p.sh[which];
    const T *x = reinterpret_cast<const T *>(which == 0 ? p.k : p.v) + (sp.t0 + lo - start + token) * st;
    const float *c_row = p.cos_table + (lo + token) * (rot >> 1) + V * u, *s_row = p.sin_table + (lo + token) * (rot >> 1) + V * u;
    __shared__ float red[3][WIDE / 32];
    uint4 raw[PASSES][2];
    auto load = [&](int h) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
            if (i * TOKENS + token < count) {
                raw[i][0] = load_stream(x + i * TOKENS * st + h * sh + at.a);
                raw[i][1] = load_stream(x + i * TOKENS * st + h * sh + at.b);
            }
    };
    load(head0);
    const int head1 = min(head0 + heads_each, (int)p.kv_heads);
#pragma unroll 1
    for (int h = head0; h < head1; ++h) {
        Pair<T> v[PASSES];
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
            if (i * TOKENS + token < count) {
                unpack(v[i].a, raw[i][0], T());
                unpack(v[i].b, raw[i][1], T());
                if (at.turns) {                                      // the rows stay in L1 from head to head
                    float c[V], s[V];
                    load_row(c, c_row + i * TOKENS * (rot >> 1));
                    load_row(s, s_row + i * TOKENS * (rot >> 1));
                    turn<T>(v[i], c, s, at);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) a = max_abs(max_abs(a, v[i].a[e]), v[i].b[e]);
            }
        if (h + 1 < head1) load(h + 1);
        uint8_t *codes = p.codes[which] + (page * p.kv_heads + h) * p.page_size * D;
        float *scale = p.scale[which] + page * p.kv_heads + h;
        const float before = held ? *scale : 0.0f;
        auto over_task = [&](float x, float *r) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x = max_abs(x, __shfl_xor_sync(0xffffffffu, x, o));
            if constexpr (TT > 32) {
                if (lane == 0) r[tid >> 5] = x;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WIDE / 32; ++w) x = max_abs(x, r[w]);
            }
            return x;
        };
        a = over_task(a, red[(h - head0) & 1]);                      // (the other one may still be read for the last head)
        const bool all_finite = a < INFINITY;
        if (!all_finite) {                                           // the scale is that of the finite values
            a = 0.0f;
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
                if (i * TOKENS + token < count)
#pragma unroll
                    for (int e = 0; e < V; ++e) a = fmaxf(a, fmaxf(finite_abs(v[i].a[e]), finite_abs(v[i].b[e])));
            a = over_task(a, red[2]);
            if constexpr (TT > 32) __syncthreads();                  // red[2] has been read
        }
        const float s = fmaxf(block_scale(a), before);
        const float inv = 1.0f / s;                                  // a power of two: exact
        if (held && s > before) {
            const float ratio = before * inv;
            for (int i = worker * 4; i < held * D; i += TT * 4) {
                uchar4 old = *reinterpret_cast<const uchar4 *>(codes + i);
                old.x = float_to_e4m3(e4m3_to_float(old.x) * ratio), old.y = float_to_e4m3(e4m3_to_float(old.y) * ratio);
                old.z = float_to_e4m3(e4m3_to_float(old.z) * ratio), old.w = float_to_e4m3(e4m3_to_float(old.w) * ratio);
                *reinterpret_cast<uchar4 *>(codes + i) = old;
            }
        }
        codes += (held + token) * D;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
            if (i * TOKENS + token < count) {
                store_codes(codes + i * TOKENS * D + at.a, v[i].a, inv, all_finite);
                store_codes(codes + i * TOKENS * D + at.b, v[i].b, inv, all_finite);
            }
        if constexpr (TT > 32) {
            if (tid == 0) *scale = s;
        } else {
            __syncwarp();                                            // every lane has read the old scale
            if (lane == 0) *scale = s;
        }
    }
}

// Whether rows can be read and written 16 bytes at a time, in pairs of pieces that rotate with one another.
bool wide_enough(const piton_kv_append_args *a, int size) {
    const int64_t v = 16 / size;
    if (a->rot_dim % (2 * v)) return false;
    uint64_t bits = a->k | a->v;
    for (int64_t s : {a->stride_kt, a->stride_kh, a->stride_vt, a->stride_vh}) bits |= (uint64_t)s * size;
    if (a->q_heads) {
        bits |= a->q | a->q_out;
        for (int64_t s : {a->stride_qt, a->stride_qh, a->stride_ot, a->stride_oh}) bits |= (uint64_t)s * size;
    }
    if (a->rot_dim) bits |= a->cos_table | a->sin_table;
    return bits % 16 == 0;
}

template <typename T, int D, int TT, int PASSES> int launch_wide(AppendParams p, cudaStream_t s) {
    constexpr int UPH = D / (2 * (16 / (int)sizeof(T))), SIDE = 32 / UPH;
    const int64_t sms = num_sms();
    // A CTA walks a unit's heads, whose rows share what it read of the rotation tables, as far as that leaves two CTAs an SM
    // (10,500 tokens at most, 32 + 32 heads of 64, fp32: 59 us; at most 4 heads a CTA 78, one 146).
    int64_t heads_each = 1;
    if (TT == WIDE) {
        heads_each = p.units * 2 * p.kv_heads / (2 * sms);
        heads_each = heads_each < 1 ? 1 : heads_each > p.kv_heads ? p.kv_heads : heads_each;
    }
    const int64_t tasks = p.units * 2 * cdiv(p.kv_heads, heads_each);
    p.unit_blocks = cdiv(tasks, WIDE / TT);
    // A warp walks a token's query heads, in pieces while there are not 8 warps an SM (64 tokens of 32 heads: 4.3 us, whole 5.2;
    // 1600 tokens: whole 8.2, in pieces up to 32 warps an SM 10.1).
    int64_t q_pieces = 1;
    while (q_pieces * SIDE < p.q_heads && p.tokens * q_pieces < 8 * sms) q_pieces *= 2;
    const int64_t blocks = p.unit_blocks + (p.q_heads ? cdiv(p.tokens * q_pieces, WIDE / 32) : 0);
    PITON_REQUIRE(blocks < (1ll << 31), "too many blocks: %lld", (long long)blocks);
    kv_append_wide_kernel<T, D, TT, PASSES><<<(unsigned)blocks, WIDE, 0, s>>>(p, (int)heads_each, (int)q_pieces);
    return check_launch("kv_append");
}

template <typename T, int D> int launch_wide(const AppendParams &p, cudaStream_t s) {
    constexpr int UPH = D / (2 * (16 / (int)sizeof(T)));
    // Pairs of a task at most: what a warp's four passes hold is a warp's, more is a CTA's (1600 tokens in pages of 16, 64
    // dimensions, bf16, 64 pairs: a warp 8.2 us, a CTA 9.1).
    const int64_t most = (p.cu || p.uniform > p.page_size ? p.page_size : p.uniform) * UPH;
    if (most <= 32) return launch_wide<T, D, 32, 1>(p, s);
    if (most <= 128) return launch_wide<T, D, 32, 4>(p, s);
    if (most <= WIDE) return launch_wide<T, D, WIDE, 1>(p, s);
    if (most <= 2 * WIDE) return launch_wide<T, D, WIDE, 2>(p, s);
    if (most <= 4 * WIDE) return launch_wide<T, D, WIDE, 4>(p, s);
    return launch_wide<T, D, WIDE, 8>(p, s);
}

}  // namespace

int kv_append_status_read_and_clear(int *status) {
    int zero = 0;
    PITON_CUDA(cudaMemcpyFromSymbol(status, g_append_status, sizeof(int)));
    PITON_CUDA(cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int)));
    return PITON_B200_OK;
}

}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

extern "C" int piton_b200_kv_append(const piton_kv_append_args *a, void *stream) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->kv_heads > 0 && a->q_heads >= 0 && a->num_pages >= 0 &&
                      a->table_width >= 0 && a->rope_len >= 0,
                  "bad shape");
    PITON_REQUIRE(a->batch < (1 << 24) && a->tokens < (1ll << 31) && a->kv_heads <= (1 << 16) && a->q_heads <= (1 << 16) &&
                      a->num_pages < (1ll << 31),
                  "batch, tokens, heads or pages beyond the 32-bit offsets");
    if ((a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) ||
        (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128))
        return set_error(PITON_B200_ENOTSUP, "head_dim %lld (32, 64, 128) or page_size %lld (16, 32, 64, 128)",
                         (long long)a->head_dim, (long long)a->page_size);
    PITON_REQUIRE(a->rot_dim >= 0 && a->rot_dim <= a->head_dim && a->rot_dim % 2 == 0, "rot_dim %lld", (long long)a->rot_dim);
    PITON_REQUIRE(a->batch > 0 || a->tokens == 0, "%lld tokens of no sequence", (long long)a->tokens);
    if (a->batch == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->cu || a->tokens % a->batch == 0, "%lld tokens are not the same number for %lld sequences",
                  (long long)a->tokens, (long long)a->batch);
    PITON_REQUIRE(a->starts && a->lengths != a->starts, "starts is NULL or the same as lengths");
    PITON_REQUIRE(a->tokens == 0 || (a->k && a->v && a->k_codes && a->v_codes && a->k_scale && a->v_scale && a->table),
                  "NULL pointer");
    PITON_REQUIRE(a->k_codes % 16 == 0 && a->v_codes % 16 == 0, "codes are not 16-byte aligned");
    PITON_REQUIRE(a->tokens == 0 || a->rot_dim == 0 || (a->cos_table && a->sin_table), "rotation tables are NULL");
    PITON_REQUIRE(a->tokens == 0 || a->q_heads == 0 || (a->q && a->q_out), "q or q_out is NULL");
    AppendParams p;
    p.k = reinterpret_cast<const void *>(a->k);
    p.v = reinterpret_cast<const void *>(a->v);
    p.q = reinterpret_cast<const void *>(a->q);
    p.q_out = reinterpret_cast<void *>(a->q_out);
    p.codes[0] = reinterpret_cast<uint8_t *>(a->k_codes);
    p.codes[1] = reinterpret_cast<uint8_t *>(a->v_codes);
    p.scale[0] = reinterpret_cast<float *>(a->k_scale);
    p.scale[1] = reinterpret_cast<float *>(a->v_scale);
    p.table = reinterpret_cast<const int32_t *>(a->table);
    p.starts = reinterpret_cast<const int32_t *>(a->starts);
    p.cu = reinterpret_cast<const int32_t *>(a->cu);
    p.lengths = reinterpret_cast<int32_t *>(a->lengths);
    p.cos_table = reinterpret_cast<const float *>(a->cos_table);
    p.sin_table = reinterpret_cast<const float *>(a->sin_table);
    p.batch = a->batch; p.tokens = a->tokens; p.kv_heads = a->kv_heads; p.q_heads = a->q_heads;
    p.page_size = a->page_size; p.num_pages = a->num_pages; p.table_width = a->table_width; p.table_stride = a->table_stride;
    p.st[0] = a->stride_kt; p.sh[0] = a->stride_kh; p.st[1] = a->stride_vt; p.sh[1] = a->stride_vh;
    p.sqt = a->stride_qt; p.sqh = a->stride_qh; p.sot = a->stride_ot; p.soh = a->stride_oh;
    p.rope_len = a->rope_len;
    p.dim = (int32_t)a->head_dim; p.rot = (int32_t)a->rot_dim; p.interleaved = a->interleaved;
    p.uniform = a->cu ? 0 : a->tokens / a->batch;
    // a run of n tokens touches at most ceil((n - 1) / page_size) + 1 pages
    p.units = a->cu ? a->tokens / a->page_size + 2 * a->batch
                    : a->batch * (p.uniform ? cdiv(p.uniform - 1, a->page_size) + 1 : 1);
    p.unit_blocks = p.units * 2 * a->kv_heads;
    const int64_t blocks = p.unit_blocks + cdiv(a->tokens * a->q_heads, THREADS / 32);
    PITON_REQUIRE(blocks < (1ll << 31), "too many blocks: %lld", (long long)blocks);
    if (wide_enough(a, a->type == PITON_B200_TYPE_F32 ? 4 : 2))
        return with_type(a->type, [&](auto t) {
            using T = decltype(t);
            cudaStream_t q = as_stream(stream);
            return p.dim == 32 ? launch_wide<T, 32>(p, q) : p.dim == 64 ? launch_wide<T, 64>(p, q) : launch_wide<T, 128>(p, q);
        });
    return with_type(a->type, [&](auto t) {
        kv_append_kernel<decltype(t)><<<(unsigned)blocks, THREADS, 0, as_stream(stream)>>>(p);
        return check_launch("kv_append");
    });
}
