// Attention of a few query tokens per sequence over the paged 8-bit cache (kv_append.cu's layout).
//
// For every row (query token, head): s_j = scale q . k_j over the keys it sees, o = sum_j softmax(s)_j v_j,
// in one pass over the keys with the running maximum and sum of the softmax.  Each key and value byte is
// read once per 16 rows, and a row tile does 4 D flops per 2 D bytes, so the cache's bytes bound it.
//
// A CTA takes up to 16 rows that share a key head (row = token * group + head of the group) and a range of keys;
// its four warps take 32 keys at a time in turn, each with its own softmax state, and never wait for one
// another before the end.  With the scores computed as S^T = K Q^T and the output as O^T = V^T P^T, keys and
// dimensions are the 16-row side of mma.m16n8k16 and the rows its 8-column side, so one query token's group of
// heads fills an instruction.  Every e4m3 code is exact in fp16: queries are scaled by a power of two per row
// and rounded to fp16 (exact for 16-bit rows down to 2^-28 of the row's largest; fp32 ones split into two halves, 22 bits down to
// 2^-17 of it).  The weights p become fp16 too: two halves, 22 bits, for fp32 rows and for fp16 ones, whose output one half's
// rounding would show in (64 sequences of 2000 keys: two halves 60 us, one 58; error against 64 bits 2.1e-4 and 2.8e-4); one, 11 bits, for bf16 rows,
// three more than the output's.  Products are exact in the fp32 accumulators.  Weights are kept as 2^LIFT p relative to a reference that may lag the running
// maximum by 2^SLACK (16-bit rows), so O is rarely rescaled and the products add straight into its registers; fp32 rows add a
// stage's sums to O in fp32 instead.  The pages' V scales go into the weights relative to a reference
// that a tile's scale passes by no more than 2^6 downwards: weights down to 2^-19 of the row's largest keep a half's 11 bits, those
// below 2^-30 are lost. The reference moves with the scales, up or down, and the sums so far move in fp32, so what a row
// adds up from pages of small values does not depend on larger ones that it does not see or hardly weighs (within 2^80 of them).
//
// The order of dimensions inside an MMA's k index is free as long as K and Q agree, so a lane copies (cp.async) the 16 bytes
// of a key row that its own fragment holds, or whole rows go into one copy where they are 128 bytes, and the same for V with
// dimension blocks: shared memory is each warp's private queue of two stages of keys and one of values (12 KB at 128 dimensions),
// read back without bank conflicts and without a barrier of the CTA.
//
// When there are fewer (sequence, key head, row tile) units than CTAs fit the GPU at once, the keys are split into ranges that
// fill one wave, and a second kernel, launched while the first finishes, joins them in a fixed order. More splits than one wave were slower
// (24 sequences, 4 new tokens, window 2048: 240 CTAs 34.3 us, 360 CTAs 45.4).
//
// Measured: 268 MB of codes, one sequence, bf16: 63 us (4.3 TB/s); 32 sequences, fp32, 538 MB: 113 us (4.8 TB/s); 64
// sequences of 2000 keys, fp16: 60.5 us (3.3 TB/s); one of 1000 keys: 8.5 us, of 100 keys and 4 heads: 4.5. Up to 8 rows a tile the copies bound it
// once a warp has several stages; with 16 rows the chain of products, softmax and products of 8 warps an SM does (34.3 us
// where the bytes take 9.8; instructions issue in 30 % of the cycles).
#include <type_traits>

#include "decode.cuh"

namespace piton {
namespace decode {

__device__ int g_cached_status = 0;

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// V scales more than 2^NEAR below their reference move it, though not 2^MOST below the largest: what has been added up stays in fp32's range.
constexpr int NEAR = 6, MOST = 80;
constexpr uint32_t BAD_PAGE = 0x7FC0DEADu;   // in a stage's scale slot: the tile's page was not followed

struct CachedParams {
    const void *q;
    void *out;
    float *lse;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *lengths, *cu;
    float *part_o;                       // [splits][tokens * q_heads][D], splits > 1 only
    float2 *part_ml;                     // [splits][tokens * q_heads]
    int64_t batch, tokens, num_pages, table_stride, sqt, sqh, sot, soh, window, uniform, chunk;
    int32_t q_heads, kv_heads, group, page_log2, table_width, row_tiles, splits, q_aligned;
    float scale;
};

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_cached_status, 0, code); }

template <int D> struct Geometry {
    static constexpr int KB = D >= 64 ? 16 : D / 4;     // bytes of a key row in one copy of a lane
    static constexpr int KC = D / (4 * KB);             // such copies per row
    static constexpr int VB = D / 8;                    // bytes of a value row that a lane takes
    static constexpr int TILES = D == 128 ? 2 : 4, KEYS = 16 * TILES;     // of a stage: 16-key tiles, each inside one page
    // a warp's queue: two stages of keys and one of values, whose copies run while the scores are computed
    static constexpr int BYTES = KEYS * D, QUEUE = 3 * BYTES, RING = WARPS * QUEUE;
    static constexpr int SCALES = 8 * TILES;            // bytes of a stage's K and V scales, tile by tile
    static constexpr int SMEM = RING + WARPS * 2 * SCALES;
    static constexpr int RUN = 32 / TILES;              // stages whose page numbers the lanes hold at a time
};

template <int N> __device__ __forceinline__ void copy_or_clear(uint32_t dst, const void *src, bool on) {
    const int size = on ? N : 0;                        // the rest of the N bytes is filled with zeros
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(size), "n"(N) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Two e4m3 codes, bytes 0 and 1 (or 2 and 3) of a word, as two fp16 values: exact.
__device__ __forceinline__ uint32_t halves(uint32_t word) {
    uint32_t d;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(word));
    return d;
}
__device__ __forceinline__ uint32_t high_halves(uint32_t word) {
    uint32_t d;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(d) : "r"(word));
    return d;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// What the fp16 halves of `packed` leave of (lo, hi), as fp16 again.
__device__ __forceinline__ uint32_t pack_rest(uint32_t packed, float lo, float hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&packed));
    return pack(lo - f.x, hi - f.y);
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // c = a b
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four elements of a row, in one load where rows are aligned for it.
template <typename T> __device__ __forceinline__ void load_four(float (&x)[4], const T *at, bool aligned) {
    T v[4];
    if (aligned) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(at);
        else *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(at);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = at[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = to_float(v[e]);
}
// The biased exponent of a positive normal number up to 2^126, 0 for anything else.
__device__ __forceinline__ int exponent(float x) {
    const uint32_t e = __float_as_uint(x) >> 23;
    return e <= 253 ? (int)e : 0;
}
__device__ __forceinline__ float power(int e) { return __int_as_float(e + 127 << 23); }      // 2^e, -126 <= e <= 127
// An exponent to move sums by as a byte, and the factor: sums that move down by more than 2^126 are none.
__device__ __forceinline__ uint32_t move_by(int e) { return (uint32_t)(max(e, -127) + 128); }
__device__ __forceinline__ float move_of(uint32_t byte) { return __uint_as_float(byte - 1 << 23); }
// NaN codes (7F and FF) of a word: a set high bit in each such byte.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// CTAs an SM holds: registers bound it. Two of 16 rows a tile at 128 dimensions or in fp32, where three spill more than they hide (24
// sequences, 4 new tokens, window 2048, fp32: 2 CTAs, which spill 264 bytes a thread, 40.0 us, 3 CTAs 57.4); three below that, which
// short sequences gain from and long ones pay for (16 bits, 64 dimensions, 230 sequences of 200 keys: 3 CTAs 47 us, 2 CTAs 57.5; 64 of
// 2000 keys: 57.6 and 51).
constexpr int ctas(int nq, int dim, bool fp32) { return nq == 1 || (dim <= 64 && !fp32) ? 3 : 2; }

// The rows of a tile that a lane holds in its score and output fragments: columns 2 j and 2 j + 1 of each of the NQ
// 8-row groups; the keys [first, pos] that each sees.
template <int NQ> struct Rows {
    int32_t first[NQ][2], pos[NQ][2];
};

// Tokens [lo, hi) of the query are those that the offsets `cu` name; the outputs of the others are those of rows that see no key.
__device__ __forceinline__ Span named(const CachedParams &p) {
    const int64_t lo = min(max((int64_t)p.cu[0], (int64_t)0), p.tokens), hi = min(max((int64_t)p.cu[p.batch], (int64_t)0), p.tokens);
    return {lo, max(hi - lo, (int64_t)0)};
}
template <typename T, int D> __device__ void clear_unnamed(const CachedParams &p, int64_t b, int kvh) {
    const Span sp = named(p);
    for (int64_t u = b; u < p.tokens - sp.n; u += p.batch) {
        const int64_t t = u < sp.t0 ? u : u + sp.n;
        for (int x = threadIdx.x; x < p.group * D; x += THREADS) {
            const int h = kvh * p.group + x / D;
            reinterpret_cast<T *>(p.out)[t * p.sot + h * p.soh + x % D] = from_float<T>(0.0f);
            if (p.lse && x % D == 0) p.lse[t * p.q_heads + h] = -INFINITY;
        }
    }
}

// The rows row0 ... of a sequence's tokens times group over one split of its keys.
template <typename T, int D, int NQ>
__device__ __forceinline__ void attend(const CachedParams &p, const int64_t b, const int kvh, const int split, const Span &sp, const uint32_t row0) {
    using G = Geometry<D>;
    constexpr bool SPLIT = sizeof(T) == 4;              // fp32 rows: queries and weights as pairs of halves
    constexpr bool PAIRS = !std::is_same_v<T, __nv_bfloat16>;   // of weights, also for fp16
    constexpr float LIFT = SPLIT ? 14.0f : 11.0f, SLACK = SPLIT ? 0.0f : 4.0f, UNLIFT = SPLIT ? 0x1p-14f : 0x1p-11f;
    constexpr int R = 8 * NQ, KW = G::KB / 4, VW = G::VB / 4, MT = D / 16, KT = D / 16, TILES = G::TILES, KEYS = G::KEYS;
    extern __shared__ __align__(16) uint8_t ring[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
    const uint32_t group = p.group, rows = (uint32_t)sp.n * group;     // below 2^31, as tokens * heads is
    const uint32_t live = min((uint32_t)R, rows - row0);
    // positions are below 2^31 (lengths are int32); a row past the tile's last repeats the last one
    const int32_t length = p.lengths[b];
    const int32_t *table = p.table + b * p.table_stride;
    const int64_t held = (int64_t)p.table_width << p.page_log2;
    // Without a window the first keys do not depend on the length, so their page numbers are read along with it.
    int32_t ahead = -1;
    if (!p.window) {
        const int64_t key = (int64_t)split * p.chunk + warp * KEYS + (int64_t)(lane / TILES) * (KEYS * WARPS) + 16 * (lane % TILES);
        if (key < held) ahead = table[key >> p.page_log2];
    }
    const int32_t before = length - (int32_t)sp.n;      // position of query token 0
    auto pos_of = [&](uint32_t r) { return before + (int32_t)((row0 + min(r, live - 1)) / group); };
    auto first_of = [&](int32_t pos) { return p.window ? (int32_t)max((int64_t)pos - p.window + 1, (int64_t)0) : 0; };
    const int32_t pos_lo = pos_of(0), pos_hi = pos_of(R - 1);
    const int32_t first_lo = first_of(pos_lo), first_hi = first_of(pos_hi);
    int64_t end = (int64_t)pos_hi + 1;                  // no row of the tile sees a key outside [first_lo, end)
    if (end > held) {
        if (threadIdx.x == 0) record_status(STATUS_BAD_POSITION);
        end = held;
    }
    const int64_t begin = (int64_t)(first_lo & ~(KEYS - 1)) + (int64_t)split * p.chunk;
    const int64_t stop = split == p.splits - 1 ? end : min(end, begin + p.chunk);
    const int64_t mine = begin + warp * KEYS;
    // From here on keys are counted from `mine`, in 32 bits: [0, span) is this warp's range, its stage s the KEYS from s STRIDE on.
    // What lies far before it is as good as just before.
    constexpr int32_t STRIDE = KEYS * WARPS;
    const int32_t span = (int32_t)max(stop - mine, (int64_t)0), mine32 = (int32_t)mine;
    const int32_t stages = span / STRIDE + (span % STRIDE != 0);
    auto from_mine = [&](int32_t pos) { return (int32_t)max((int64_t)pos - mine, (int64_t)-1); };
    const int32_t lo = from_mine(first_lo), lo_all = from_mine(first_hi), hi_all = from_mine(pos_lo);    // every row sees [lo_all, hi_all]

    // ---- this lane's copies ----
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(ring) + warp * G::QUEUE;
    const uint32_t scales0 = (uint32_t)__cvta_generic_to_shared(ring) + G::RING + warp * (2 * G::SCALES);
    const int32_t page_mask = (1 << p.page_log2) - 1;
    // Keys: copy i of a tile's 2 KC takes rows k_row + k_step i, a lane 16 (8) bytes. At 128 bytes a row, whole rows go into one
    // copy (half rows, each lane its own fragment, reach 5.2 TB/s where whole ones reach 6.4) and odd rows' halves are
    // exchanged, so that the fragments' reads meet no bank conflicts; below that a lane copies what it will read.
    constexpr int K_STEP = G::KC == 2 ? 4 : 8;
    const int k_row = G::KC == 2 ? lane >> 3 : g;
    const uint32_t k_slot = ring0 + (G::KC == 2 ? k_row * D + ((lane & 7) ^ (k_row & 1) << 2) * 16 : lane * G::KB);
    const uint32_t k_read[2] = {ring0 + (G::KC == 2 ? g * D + (j + 4 * (g & 1)) * 16 : lane * G::KB),
                                ring0 + (G::KC == 2 ? g * D + (j + 4 * (~g & 1)) * 16 : lane * G::KB)};
    const uint32_t v_slot = ring0 + 2 * G::BYTES + lane * G::VB;
    const uint32_t head_bytes = (uint32_t)D << p.page_log2, page_bytes = head_bytes * p.kv_heads;     // below 2^31 (heads are below 2^16)
    const uint8_t *k_lane = p.kc + (int64_t)kvh * head_bytes + k_row * D + (G::KC == 2 ? (lane & 7) * 16 : j * G::KB);
    const uint8_t *v_lane = p.vc + (int64_t)kvh * head_bytes + 2 * j * D + g * G::VB;
    int32_t ids = -1, ids_next = -1, ids_v = -1;        // pages of the 32 tiles of RUN stages, lane by lane; the values' are a stage behind
    uint32_t off_run = 0, off_run_v = 0;                // which of them are not to be read
    auto load_ids = [&](int s0) {                       // stages s0 .. s0 + RUN - 1
        const uint32_t at = (uint32_t)(s0 + lane / TILES) * STRIDE + 16 * (lane % TILES);       // may pass 2^31
        if (at >= (uint32_t)span || (int32_t)at < lo - 15) return -1;
        const int32_t id = s0 == 0 && !p.window ? ahead : table[(mine32 + (int32_t)at) >> p.page_log2];
        if (id >= 0 && id < p.num_pages) return id;
        record_status(STATUS_BAD_PAGE);
        return -1;
    };
    auto whole = [&](int32_t at, int s, uint32_t off) { // every key of the stage exists
        return at >= lo && span - at >= KEYS && !(off >> (TILES * (s % G::RUN)) & ((1u << TILES) - 1));
    };
    auto row_of = [&](const uint8_t *lane_at, int32_t id, int32_t at) {     // of a lane's first key in a tile
        return lane_at + (uint64_t)(uint32_t)max(id, 0) * page_bytes + (uint32_t)((mine32 + at & page_mask) * D);
    };
    auto issue_k = [&](int s) {
        if (s < stages) {
            if (s % G::RUN == 0) {
                ids = s == 0 ? load_ids(0) : ids_next;
                off_run = __ballot_sync(0xffffffffu, ids < 0);
                ids_next = load_ids(s + G::RUN);
            }
            const int32_t key0 = s * STRIDE;
            const uint32_t at = k_slot + (s & 1) * G::BYTES;
            const bool all = whole(key0, s, off_run);
            if (all) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint8_t *src = row_of(k_lane, __shfl_sync(0xffffffffu, ids, TILES * (s % G::RUN) + t), key0 + 16 * t);
#pragma unroll
                    for (int i = 0; i < 2 * G::KC; ++i)
                        copy_async<G::KB>(at + (2 * t * G::KC + i) * 32 * G::KB, src + i * K_STEP * D);
                }
            } else {
#pragma unroll 1
                for (int t = 0; t < TILES; ++t) {
                    const int32_t id = __shfl_sync(0xffffffffu, ids, TILES * (s % G::RUN) + t);
                    const int32_t key = key0 + 16 * t;
                    const uint8_t *src = row_of(k_lane, id, key);
#pragma unroll
                    for (int i = 0; i < 2 * G::KC; ++i) {
                        const int row = k_row + i * K_STEP;
                        const bool on = id >= 0 && key + row >= lo && key < span - row;
                        copy_or_clear<G::KB>(at + (2 * t * G::KC + i) * 32 * G::KB, on ? src + i * K_STEP * D : p.kc, on);
                    }
                }
            }
            // lane 2 t: tile t's K scale, lane 2 t + 1: its V scale
            const int32_t id = __shfl_sync(0xffffffffu, ids, TILES * (s % G::RUN) + (lane >> 1) % TILES);
            if (lane < 2 * TILES) {
                const uint32_t to = scales0 + (s & 1) * G::SCALES + lane * 4;
                if (id >= 0) copy_async<4>(to, (lane & 1 ? p.vs : p.ks) + ((int64_t)id * p.kv_heads + kvh));
                else asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(BAD_PAGE) : "memory");
            }
        }
        commit();
    };
    auto issue_v = [&](int s) {
        if (s < stages) {
            if (s % G::RUN == 0) ids_v = ids, off_run_v = off_run;     // the keys are at most one stage on
            const int32_t key0 = s * STRIDE;
            const uint32_t at = v_slot;
            const bool all = whole(key0, s, off_run_v);
            if (all) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint8_t *src = row_of(v_lane, __shfl_sync(0xffffffffu, ids_v, TILES * (s % G::RUN) + t), key0 + 16 * t);
#pragma unroll
                    for (int r = 0; r < 4; ++r)             // rows 2 j + (r & 1) + 8 (r >> 1)
                        copy_async<G::VB>(at + (4 * t + r) * 32 * G::VB, src + ((r & 1) + 8 * (r >> 1)) * D);
                }
            } else {
#pragma unroll 1
                for (int t = 0; t < TILES; ++t) {
                    const int32_t id = __shfl_sync(0xffffffffu, ids_v, TILES * (s % G::RUN) + t);
                    const int32_t key = key0 + 16 * t;
                    const uint8_t *src = row_of(v_lane, id, key);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 2 * j + (r & 1) + 8 * (r >> 1);
                        const bool on = id >= 0 && key + row >= lo && key < span - row;
                        copy_or_clear<G::VB>(at + (4 * t + r) * 32 * G::VB, on ? src + ((r & 1) + 8 * (r >> 1)) * D : p.vc, on);
                    }
                }
            }
        }
        commit();
    };
    issue_k(0);
    issue_k(1);
    issue_v(0);

    // ---- the queries: B fragments, scaled by a power of two per row ----
    uint32_t qh[NQ][KT][2], ql[SPLIT ? NQ : 1][KT][2];
    float factor[NQ][2];                                // scale * log2(e) / (the row's power of two)
    Rows<NQ> seen;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const uint32_t r = row0 + min((uint32_t)(8 * n + g), live - 1);
        const T *q = reinterpret_cast<const T *>(p.q) + (sp.t0 + r / group) * p.sqt + (kvh * group + r % group) * p.sqh;
        float x[KT][4], top = 0.0f;
#pragma unroll
        for (int k = 0; k < KT; ++k) load_four(x[k], q + (k / KW) * 64 + j * G::KB + 4 * (k % KW), p.q_aligned);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, isfinite(x[k][e]) ? fabsf(x[k][e]) : 0.0f);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's largest magnitude in [2^14, 2^15)
        const int up = top == 0.0f ? 0 : min(max(14 + 127 - (int)(__float_as_uint(top) >> 23), -112), 112);
        const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float lo = x[k][2 * e] * f, hi = x[k][2 * e + 1] * f;
                qh[n][k][e] = pack(lo, hi);
                if constexpr (SPLIT) ql[n][k][e] = pack_rest(qh[n][k][e], lo, hi);
            }
        const float own = p.scale * LOG2E * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            factor[n][e] = __shfl_sync(0xffffffffu, own, 4 * (2 * j + e));
            seen.pos[n][e] = pos_of(8 * n + 2 * j + e);
            seen.first[n][e] = first_of(seen.pos[n][e]);
        }
    }

    float o[MT][NQ][4], m[NQ][2], l[NQ][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.0f;
    // O (fp32 rows: a stage's sums) is kept relative to a power of two that the tiles' V scales lie close below: its exponent as in the bits of
    // a float, 0 before the first, and the largest it has been.
    int vref = 0, vmax = 0;

#pragma unroll 1
    for (int s = 0; s < stages; ++s) {
        const int32_t key0 = s * STRIDE;
        const uint32_t at = (s & 1) * G::BYTES;
        wait<2>();                                      // the next stage's keys and this one's values may be on their way
        __syncwarp();                                   // copies of other lanes
        float kscale[TILES], weight[TILES];
        int vtop = 0, vlow = 255;
        uint32_t bad = 0;                               // tiles whose page was not followed
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            uint32_t sc[2];
            load_words(sc, scales0 + (s & 1) * G::SCALES + 8 * t);
            bad |= (uint32_t)(sc[0] == BAD_PAGE) << t;
            kscale[t] = __uint_as_float(sc[0]);
            weight[t] = sc[0] == BAD_PAGE ? 0.0f : __uint_as_float(sc[1]);
            const int e = exponent(weight[t]);
            if (e > 0) vtop = max(vtop, e), vlow = min(vlow, e);
        }
        // The tiles' V scales relative to the reference go into the weights. It moves, and what has been added up with it, when a tile's
        // scale is above it or too far below for fp16.
        uint32_t moves = 0;                             // byte t: 128 more than the exponent that the sums move by before tile t, 0: they do not
        const int rtop = SPLIT ? vtop : max(vtop, vref);
        bool level = true;
        if (vlow >= rtop - NEAR) {                      // close together (or no scale at all)
            if (!SPLIT && vref && rtop > vref) moves = move_by(vref - rtop);
            vref = rtop;
            vmax = max(vmax, vref);
#pragma unroll
            for (int t = 0; t < TILES; ++t) level = level && __float_as_int(weight[t]) == vref << 23;
            if (!level && vref) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) weight[t] *= power(127 - vref);
            }
            level = level && vref;                      // without a reference the weights are the scales: zeros, or not numbers
        } else {
            level = false;
            if (SPLIT) vref = vmax = 0;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const int e = exponent(weight[t]), next = !e ? vref : e > vref ? e : e < vref - NEAR ? max(e, vmax - MOST) : vref;
                if (vref && next != vref) moves |= move_by(vref - next) << (8 * t);
                vref = next;
                vmax = max(vmax, next);
                if (vref) weight[t] *= power(127 - vref);
            }
        }

        // ---- scores ----
        float c[TILES][NQ][4];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
#pragma unroll
            for (int h = 0; h < G::KC; ++h) {
                uint32_t w0[KW], w1[KW];
                load_words(w0, k_read[h] + at + 2 * t * G::KC * 32 * G::KB);             // row g
                load_words(w1, k_read[h] + at + (2 * t + 1) * G::KC * 32 * G::KB);       // row g + 8
#pragma unroll
                for (int k = 0; k < KW; ++k) {
                    const uint32_t a[4] = {halves(w0[k]), halves(w1[k]), high_halves(w0[k]), high_halves(w1[k])};
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        if (h + k == 0) mma_first(c[t][n], a, qh[n][0][0], qh[n][0][1]);
                        else mma(c[t][n], a, qh[n][h * KW + k][0], qh[n][h * KW + k][1]);
                        if constexpr (SPLIT) mma(c[t][n], a, ql[n][h * KW + k][0], ql[n][h * KW + k][1]);
                    }
                }
            }
        }
        __syncwarp();
        issue_k(s + 2);

        // ---- softmax ----
        const bool edge = key0 < lo_all || key0 > hi_all - (KEYS - 1) || span - key0 < KEYS || bad;
        uint32_t off[NQ];
        float alpha[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[t][n][e] = c[t][n][e] * factor[n][e & 1] * kscale[t];
            off[n] = 0;                                 // bit 4 t + e: this score's key is not seen by its row
            if (edge) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t in = 16 * t + g + 8 * (e >> 1), key = (int32_t)((uint32_t)(mine32 + key0) + in);     // (past 2^31: off)
                        const bool on = !(bad >> t & 1) && key0 < span - in && key >= seen.first[n][e & 1] && key <= seen.pos[n][e & 1];
                        if (!on) off[n] |= 1u << (4 * t + e), c[t][n][e] = -INFINITY;
                    }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = fmaxf(c[0][n][e], c[0][n][e + 2]);
#pragma unroll
                for (int t = 1; t < TILES; ++t) top = fmaxf(top, fmaxf(c[t][n][e], c[t][n][e + 2]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                // The reference of the exponents: the largest score so far; 16-bit rows let a score pass it by up to 2^SLACK, so
                // that O is rarely rescaled, which LIFT leaves room for in the weights' fp16.
                const float now = SPLIT ? fmaxf(m[n][e], top) : top - m[n][e] > SLACK ? top : m[n][e];
                const float ref = now == -INFINITY ? 0.0f : now;
                alpha[n][e] = now == m[n][e] ? 1.0f : ex2(m[n][e] - now);
                m[n][e] = now;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int x = e; x < 4; x += 2) {
                        c[t][n][x] = ex2(c[t][n][x] - ref + LIFT);  // (ref - LIFT could be rounded to less, and the weight pass fp16)
                        sum += c[t][n][x];
                    }
                l[n][e] = l[n][e] * alpha[n][e] + sum;
            }
            if (!level) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[t][n][e] *= weight[t];
            }
            if (edge) {                                 // a scale that is NaN reaches only the rows that see its keys
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (off[n] >> (4 * t + e) & 1) c[t][n][e] = 0.0f;
            }
        }

        // ---- values ----
        wait<1>();                                      // the keys after the next may be on their way
        float acc[SPLIT ? MT : 1][NQ][4];               // fp32 rows: a stage's sums, added to O in fp32
        if constexpr (!SPLIT) {
            const float shrink = moves & 255 ? move_of(moves & 255) : 1.0f;
            bool moved = moves & 255;
#pragma unroll
            for (int n = 0; n < NQ; ++n) moved = moved || alpha[n][0] != 1.0f || alpha[n][1] != 1.0f;
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][n][e] *= alpha[n][e & 1] * shrink;
            }
        }
        // A fragments of the m-tiles 2 w and 2 w + 1 (dimensions g VB + 4 w ... + 3) from a word of four keys
        auto fragments = [](uint32_t (&a)[2][4], uint32_t k0, uint32_t k1, uint32_t k8, uint32_t k9) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = __byte_perm(k0, k1, i ? 0x7362 : 0x5140), y = __byte_perm(k8, k9, i ? 0x7362 : 0x5140);
                a[i][0] = halves(x), a[i][1] = high_halves(x), a[i][2] = halves(y), a[i][3] = high_halves(y);
            }
        };
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            uint32_t v[4][VW], ph[NQ][2], pl[PAIRS ? NQ : 1][2];
#pragma unroll
            for (int r = 0; r < 4; ++r) load_words(v[r], v_slot + (4 * t + r) * 32 * G::VB);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t hi = pack(c[t][n][2 * e], c[t][n][2 * e + 1]);
                    ph[n][e] = transposed(hi);
                    if constexpr (PAIRS) pl[n][e] = transposed(pack_rest(hi, c[t][n][2 * e], c[t][n][2 * e + 1]));
                }
            if (edge) {                                 // NaN codes: 0 * NaN must not reach a row that does not see the key
                uint32_t any = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int w = 0; w < VW; ++w) any |= nan_codes(v[r][w]);
                if (__any_sync(0xffffffffu, any != 0)) {    // count the NaN that each row sees, then take the codes as zeros
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        uint32_t one[4], a[2][4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            one[r] = (nan_codes(v[r][w]) >> 7) * 0x38u;    // e4m3's 1.0
                            v[r][w] &= ~((nan_codes(v[r][w]) >> 7) * 0xFFu);
                        }
                        fragments(a, one[0], one[1], one[2], one[3]);
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            const uint32_t seen_by = ~off[n] >> (4 * t);
                            const uint32_t s0 = transposed((seen_by & 1 ? 0x3C00u : 0u) | (seen_by & 2 ? 0x3C000000u : 0u));
                            const uint32_t s1 = transposed((seen_by & 4 ? 0x3C00u : 0u) | (seen_by & 8 ? 0x3C000000u : 0u));
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float count[4] = {};
                                mma(count, a[i], s0, s1);
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (count[e] != 0.0f) o[2 * w + i][n][e] = __int_as_float(0x7FC00000);
                            }
                        }
                    }
                }
            }
            if (t > 0 && moves >> (8 * t) & 255) {
                const float move = move_of(moves >> (8 * t) & 255);
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (SPLIT) acc[i][n][e] *= move;
                            else o[i][n][e] *= move;
                        }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                uint32_t a[2][4];
                fragments(a, v[0][w], v[1][w], v[2][w], v[3][w]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        if constexpr (SPLIT) {
                            if (t == 0) mma_first(acc[2 * w + i][n], a[i], ph[n][0], ph[n][1]);
                            else mma(acc[2 * w + i][n], a[i], ph[n][0], ph[n][1]);
                            mma(acc[2 * w + i][n], a[i], pl[n][0], pl[n][1]);
                        } else {
                            mma(o[2 * w + i][n], a[i], ph[n][0], ph[n][1]);
                            if constexpr (PAIRS) mma(o[2 * w + i][n], a[i], pl[n][0], pl[n][1]);
                        }
                    }
            }
        }
        if constexpr (SPLIT) {
            const float back = (vref ? power(vref - 127) : 1.0f) * UNLIFT;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][n][e] = fmaf(o[i][n][e], alpha[n][e & 1], acc[i][n][e] * back);
        }
        issue_v(s + 1);
    }
    wait<0>();

    // ---- join the warps ----
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[n][e] *= UNLIFT;
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
        }
    __syncthreads();                                    // the queues are free
    float *so = reinterpret_cast<float *>(ring);        // [WARPS][R][D], then [WARPS][R] of (m, l)
    float2 *sml = reinterpret_cast<float2 *>(so + WARPS * R * D);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + 2 * j + e;
            if (g == 0) sml[warp * R + r] = make_float2(m[n][e], l[n][e]);
            const float back = SPLIT ? 1.0f : (vref ? power(vref - 127) : 1.0f) * UNLIFT;
            float *to = so + (warp * R + r) * D + g * G::VB;
#pragma unroll
            for (int i = 0; i < MT; ++i) *reinterpret_cast<float2 *>(to + 2 * i) = make_float2(o[i][n][e] * back, o[i][n][e + 2] * back);
        }
    __syncthreads();
    for (int x = threadIdx.x; x < (int)live * D; x += THREADS) {
        const int r = x / D, d = x % D;
        float top = -INFINITY, total = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sml[w * R + r].x);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float2 ml = sml[w * R + r];
            if (ml.y == 0.0f) continue;                 // saw no key
            const float f = ex2(ml.x - top);
            total += ml.y * f;
            sum += so[(w * R + r) * D + d] * f;
        }
        const int64_t t = sp.t0 + (row0 + r) / group, h = kvh * group + (row0 + r) % group;
        if (p.splits == 1) {
            reinterpret_cast<T *>(p.out)[t * p.sot + h * p.soh + d] = from_float<T>(total == 0.0f ? 0.0f : sum / total);
            if (p.lse && d == 0) p.lse[t * p.q_heads + h] = total == 0.0f ? -INFINITY : (top + log2f(total)) * LN2;
        } else {
            const int64_t at = (int64_t)split * p.tokens * p.q_heads + t * p.q_heads + h;
            p.part_o[at * D + d] = sum;
            if (d == 0) p.part_ml[at] = make_float2(top, total);
        }
    }
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(THREADS, ctas(NQ, D, sizeof(T) == 4)) kv_attention_kernel(const CachedParams p) {
    constexpr uint32_t R = 8 * NQ;
    if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;");    // the join may take its place, and waits
    const int64_t b = blockIdx.z;
    const int kvh = blockIdx.y, tile = blockIdx.x % p.row_tiles, split = blockIdx.x / p.row_tiles;
    const Span sp = span_of(p.cu, b, p.uniform, p.tokens);
    if (p.cu && p.splits == 1 && tile == 0) clear_unnamed<T, D>(p, b, kvh);
    // (more tiles than the launch was sized for, by too small a bound of the query tokens, are taken in turn)
    const uint32_t rows = (uint32_t)sp.n * p.group;
#pragma unroll 1
    for (uint32_t row0 = tile * R; row0 < rows; row0 += p.row_tiles * R) {
        if (row0 != tile * R) __syncthreads();          // the last tile's sums have been read
        attend<T, D, NQ>(p, b, kvh, split, sp, row0);
    }
}

// Joins a few (up to 32) splits of the keys: a warp per row, lane s holds split s's maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) kv_attention_join_few_kernel(const CachedParams p) {
    constexpr int E = D / 32, HELD = 8;                 // elements of a lane, splits that are on their way at a time
    const int lane = threadIdx.x & 31;
    const int64_t rows = p.tokens * p.q_heads, row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int64_t t = row / p.q_heads, h = row % p.q_heads;
    T *out = reinterpret_cast<T *>(p.out) + t * p.sot + h * p.soh + lane * E;
    if (p.cu) {                                         // a token of no sequence: the splits have nothing of it
        const Span sp = named(p);
        if (t < sp.t0 || t >= sp.t0 + sp.n) {
#pragma unroll
            for (int e = 0; e < E; ++e) out[e] = from_float<T>(0.0f);
            if (p.lse && lane == 0) p.lse[row] = -INFINITY;
            return;
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits' results are there
    const float2 ml = lane < p.splits ? p.part_ml[lane * rows + row] : make_float2(-INFINITY, 0.0f);
    const float *from = p.part_o + row * D + lane * E;
    float held[HELD][E];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (s0 + i >= p.splits) break;
            const float *at = from + (s0 + i) * rows * D;
            if constexpr (E == 4) *reinterpret_cast<float4 *>(held[i]) = *reinterpret_cast<const float4 *>(at);
            else if constexpr (E == 2) *reinterpret_cast<float2 *>(held[i]) = *reinterpret_cast<const float2 *>(at);
            else held[i][0] = *at;
        }
    };
    load(0);
    float top = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float factor = ml.y == 0.0f ? 0.0f : ex2(ml.x - top);
    float total = ml.y == 0.0f ? 0.0f : ml.y * factor, sum[E] = {};
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    for (int s0 = 0; s0 < p.splits; s0 += HELD) {
        if (s0) load(s0);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (s0 + i >= p.splits) break;
            const float f = __shfl_sync(0xffffffffu, factor, s0 + i);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += held[i][e] * f;   // (a NaN stays one when its weight is 0)
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = from_float<T>(total == 0.0f ? 0.0f : sum[e] / total);
    if (p.lse && lane == 0) p.lse[row] = total == 0.0f ? -INFINITY : (top + log2f(total)) * LN2;
}

// Joins more of them: a CTA per row, its warps a split in four each.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) kv_attention_join_kernel(const CachedParams p) {
    constexpr int E = D / 32;
    extern __shared__ __align__(16) float factor[];     // [splits]; then [WARPS][D] sums
    __shared__ float red[2][WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t rows = p.tokens * p.q_heads, row = blockIdx.x;
    float *sums = factor + p.splits;
    const int64_t t = row / p.q_heads, h = row % p.q_heads;
    T *out = reinterpret_cast<T *>(p.out) + t * p.sot + h * p.soh;
    if (p.cu) {                                         // a token of no sequence: the splits have nothing of it
        const Span sp = named(p);
        if (t < sp.t0 || t >= sp.t0 + sp.n) {
            if (threadIdx.x < D) out[threadIdx.x] = from_float<T>(0.0f);
            if (p.lse && threadIdx.x == 0) p.lse[row] = -INFINITY;
            return;
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits' results are there
    // up to 16 splits a warp are on their way while the factors are found
    constexpr int HELD = 16;
    float held[HELD][E];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int s = warp + WARPS * i;
#pragma unroll
        for (int e = 0; e < E; ++e) held[i][e] = s < p.splits ? p.part_o[(s * rows + row) * D + lane * E + e] : 0.0f;
    }
    float top = -INFINITY, total = 0.0f;
    for (int s = threadIdx.x; s < p.splits; s += THREADS) top = fmaxf(top, p.part_ml[s * rows + row].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[0][w]);
    for (int s = threadIdx.x; s < p.splits; s += THREADS) {
        const float2 ml = p.part_ml[s * rows + row];
        const float f = ml.y == 0.0f ? 0.0f : ex2(ml.x - top);
        factor[s] = f;
        total += ml.y == 0.0f ? 0.0f : ml.y * f;
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    if (lane == 0) red[1][warp] = total;
    __syncthreads();
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += red[1][w];
    float sum[E] = {};
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int s = warp + WARPS * i;
        const float f = s < p.splits ? factor[s] : 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += held[i][e] * f;   // (a NaN stays one when its weight is 0)
    }
#pragma unroll 4
    for (int s = warp + WARPS * HELD; s < p.splits; s += WARPS) {
        const float f = factor[s];
        const float *from = p.part_o + (s * rows + row) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += from[e] * f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[warp * D + lane * E + e] = sum[e];
    __syncthreads();
    if (threadIdx.x < D) {
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) all += sums[w * D + threadIdx.x];
        out[threadIdx.x] = from_float<T>(total == 0.0f ? 0.0f : all / total);
    }
    if (p.lse && threadIdx.x == 0) p.lse[row] = total == 0.0f ? -INFINITY : (top + log2f(total)) * LN2;
}

// How a call is cut: NQ 8-row groups a tile, row tiles a (sequence, key head), splits of the keys.
struct Plan {
    int nq;
    int64_t row_tiles, splits, chunk;
};

Plan plan_of(const piton_kv_attention_args *a) {
    Plan plan;
    const int64_t most_new = !a->cu ? a->tokens / a->batch : a->max_new && a->max_new < a->tokens ? a->max_new : a->tokens;
    const int64_t rows = most_new * (a->q_heads / a->kv_heads);
    plan.nq = rows <= 8 ? 1 : 2;
    plan.row_tiles = cdiv(rows, 8 * plan.nq);
    // keys that a row tile can see, as far as the host knows
    int64_t span = a->max_length ? a->max_length : a->table_width * a->page_size;
    span = span < a->table_width * a->page_size ? span : a->table_width * a->page_size;
    const int64_t keys = a->head_dim == 128 ? 32 : 64;  // of a stage
    if (a->window && a->window + most_new + keys < span) span = a->window + most_new + keys;
    // enough CTAs for every SM and no split below 256 keys
    const int64_t units = plan.row_tiles * a->kv_heads * a->batch, slots = (int64_t)num_sms() * ctas(plan.nq, (int)a->head_dim, a->type == PITON_B200_TYPE_F32);
    int64_t splits = units >= slots ? 1 : slots / units;
    const int64_t most = cdiv(span, 256);
    splits = splits < most ? splits : most;
    if (splits < 1) splits = 1;
    plan.chunk = cdiv(cdiv(span, splits), keys * WARPS) * (keys * WARPS);
    if (plan.chunk == 0) plan.chunk = keys * WARPS;
    plan.splits = span > 0 ? cdiv(span, plan.chunk) : 1;
    return plan;
}

template <typename T, int D, int NQ> int launch(const CachedParams &p, int64_t batch, cudaStream_t s) {
    using G = Geometry<D>;
    static_assert(WARPS * 8 * NQ * (D * 4 + 8) <= G::RING, "the warps' results fit the queues");
    static bool known[64];
    int dev = 0;
    PITON_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !known[dev]) {
        PITON_CUDA(cudaFuncSetAttribute(kv_attention_kernel<T, D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
        if (dev >= 0 && dev < 64) known[dev] = true;
    }
    const dim3 grid((unsigned)(p.row_tiles * p.splits), (unsigned)p.kv_heads, (unsigned)batch);
    kv_attention_kernel<T, D, NQ><<<grid, THREADS, G::SMEM, s>>>(p);
    if (p.splits == 1) return check_launch("kv_attention");
    // launched while the splits finish (programmatic dependent launch); it waits for them before it reads
    cudaLaunchConfig_t cfg = {};
    const int64_t rows = p.tokens * p.q_heads;
    // a warp a row for few splits (2 splits of 1920 rows: 34.3 us a call, a CTA a row 40.2), a CTA a row for more (16 splits of 32
    // rows: 9.3 us, a warp a row 9.6), unless there are many rows (13 splits of 128 rows: a warp a row 13.6, a CTA 14.0)
    const bool few = p.splits <= (rows < 128 ? 8 : 16);
    cfg.gridDim = dim3((unsigned)(few ? cdiv(rows, WARPS) : rows));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = few ? 0 : (size_t)(p.splits + WARPS * D) * sizeof(float);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PITON_CUDA(cudaLaunchKernelEx(&cfg, few ? kv_attention_join_few_kernel<T, D> : kv_attention_join_kernel<T, D>, p));
    return check_launch("kv_attention", 2);
}

template <typename T, int D> int launch(const CachedParams &p, int nq, int64_t batch, cudaStream_t s) {
    return nq == 1 ? launch<T, D, 1>(p, batch, s) : launch<T, D, 2>(p, batch, s);
}

}  // namespace

int kv_attention_status_read_and_clear(int *status) {
    int zero = 0;
    PITON_CUDA(cudaMemcpyFromSymbol(status, g_cached_status, sizeof(int)));
    PITON_CUDA(cudaMemcpyToSymbol(g_cached_status, &zero, sizeof(int)));
    return PITON_B200_OK;
}

}  // namespace decode
}  // namespace piton

using namespace piton;
using namespace piton::decode;

namespace {

int check_attention(const piton_kv_attention_args *a) {
    PITON_REQUIRE(a != nullptr, "args is NULL");
    PITON_REQUIRE(a->flags == 0, "unknown flags 0x%x", a->flags);
    PITON_REQUIRE(a->type >= PITON_B200_TYPE_F32 && a->type <= PITON_B200_TYPE_BF16, "unknown element type %d", a->type);
    PITON_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->kv_heads > 0 && a->q_heads > 0 && a->num_pages >= 0 &&
                      a->table_width >= 0 && a->window >= 0 && a->max_length >= 0 && a->max_new >= 0,
                  "bad shape");
    PITON_REQUIRE(a->q_heads % a->kv_heads == 0, "%lld query heads over %lld key heads", (long long)a->q_heads,
                  (long long)a->kv_heads);
    PITON_REQUIRE(a->batch <= 65535 && a->tokens < (1ll << 31) && a->q_heads <= 65535 && a->num_pages < (1ll << 31) &&
                      a->table_width < (1ll << 31),
                  "batch, tokens, heads or pages too large");
    if ((a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) ||
        (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128))
        return set_error(PITON_B200_ENOTSUP, "head_dim %lld (32, 64, 128) or page_size %lld (16, 32, 64, 128)",
                         (long long)a->head_dim, (long long)a->page_size);
    PITON_REQUIRE(a->batch > 0 || a->tokens == 0, "%lld tokens of no sequence", (long long)a->tokens);
    PITON_REQUIRE(a->batch == 0 || a->cu || a->tokens % a->batch == 0, "%lld tokens are not the same number for %lld sequences",
                  (long long)a->tokens, (long long)a->batch);
    return PITON_B200_OK;
}

}  // namespace

extern "C" size_t piton_b200_kv_attention_workspace_size(const piton_kv_attention_args *a) {
    if (check_attention(a) != PITON_B200_OK || a->batch == 0 || a->tokens == 0) return 0;
    const Plan plan = plan_of(a);
    return plan.splits == 1 ? 0 : (size_t)(plan.splits * a->tokens * a->q_heads) * (a->head_dim + 2) * sizeof(float);
}

extern "C" int piton_b200_kv_attention(const piton_kv_attention_args *a, void *stream) {
    if (int rc = check_attention(a)) return rc;
    if (a->batch == 0 || a->tokens == 0) return PITON_B200_OK;
    PITON_REQUIRE(a->q && a->out && a->k_codes && a->v_codes && a->k_scale && a->v_scale && a->table && a->lengths,
                  "NULL pointer");
    PITON_REQUIRE(a->k_codes % 16 == 0 && a->v_codes % 16 == 0, "codes are not 16-byte aligned");
    const Plan plan = plan_of(a);
    const int64_t rows = a->tokens * a->q_heads;
    const uint64_t need = plan.splits == 1 ? 0 : (uint64_t)(plan.splits * rows) * (a->head_dim + 2) * sizeof(float);
    if (need && (!a->workspace || a->workspace_bytes < need))
        return set_error(PITON_B200_EWORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)a->workspace_bytes,
                         (unsigned long long)need);
    PITON_REQUIRE(a->workspace % 16 == 0 || !need, "workspace is not 16-byte aligned");
    PITON_REQUIRE(plan.row_tiles * plan.splits < (1ll << 31) && rows < (1ll << 31), "tokens times heads too large");
    CachedParams p;
    p.q = reinterpret_cast<const void *>(a->q);
    p.out = reinterpret_cast<void *>(a->out);
    p.lse = reinterpret_cast<float *>(a->lse);
    p.kc = reinterpret_cast<const uint8_t *>(a->k_codes);
    p.vc = reinterpret_cast<const uint8_t *>(a->v_codes);
    p.ks = reinterpret_cast<const float *>(a->k_scale);
    p.vs = reinterpret_cast<const float *>(a->v_scale);
    p.table = reinterpret_cast<const int32_t *>(a->table);
    p.lengths = reinterpret_cast<const int32_t *>(a->lengths);
    p.cu = reinterpret_cast<const int32_t *>(a->cu);
    p.part_o = reinterpret_cast<float *>(a->workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + plan.splits * rows * a->head_dim);
    p.batch = a->batch; p.tokens = a->tokens; p.num_pages = a->num_pages; p.table_stride = a->table_stride;
    p.sqt = a->stride_qt; p.sqh = a->stride_qh; p.sot = a->stride_ot; p.soh = a->stride_oh;
    p.window = a->window; p.uniform = a->cu ? 0 : a->tokens / a->batch; p.chunk = plan.chunk;
    p.q_heads = (int32_t)a->q_heads; p.kv_heads = (int32_t)a->kv_heads; p.group = p.q_heads / p.kv_heads;
    p.page_log2 = a->page_size == 16 ? 4 : a->page_size == 32 ? 5 : a->page_size == 64 ? 6 : 7;
    p.table_width = (int32_t)a->table_width; p.row_tiles = (int32_t)plan.row_tiles; p.splits = (int32_t)plan.splits;
    p.scale = (float)a->sm_scale;
    const uint64_t size = a->type == PITON_B200_TYPE_F32 ? 4 : 2;
    p.q_aligned = (a->q | (uint64_t)a->stride_qt * size | (uint64_t)a->stride_qh * size) % (4 * size) == 0;
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        cudaStream_t s = as_stream(stream);
        if (a->head_dim == 32) return launch<T, 32>(p, plan.nq, a->batch, s);
        if (a->head_dim == 64) return launch<T, 64>(p, plan.nq, a->batch, s);
        return launch<T, 128>(p, plan.nq, a->batch, s);
    });
}
