// Attention of one new token per sequence over the pages of a cache (mni_paged_cache_attend).
#include <limits.h>

#include "lanes.h"
#include "paged_cache.h"

namespace mni {
namespace {

constexpr int TPB = 256;
constexpr float LOG2E = 1.44269504088896340736f;
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <class V>
__device__ __forceinline__ V stream(const V *p) { return __builtin_nontemporal_load(p); }

// ---- attention of one new token ------------------------------------------------------------------------------------
// softmax(scale q k^T) v by the running maximum and sum, one pass over the rows.  A workgroup takes a chunk of one
// sequence's positions for one key head; its four wavefronts walk it in tiles, each with a maximum, sum and output of its
// own.  States meet at the end, through LDS and (more than one chunk) in paged_join_kernel, always in the same order.
// Scores are kept in units of log2 e: the exponential is one v_exp_f32.  Rows are read past the caches' retention
// (nontemporal): a decoding step comes back to a row after everything else the model holds, and 1 GB of fp32 rows is read
// at 6.6 TB/s so, at 5.9 otherwise (79 MB that a benchmark finds in the last-level cache again: 21.5 us, 20.8 otherwise).
//
// paged_attend_kernel is the vector form, for any head_dim and page: one query head, LPR lanes hold a row in 16-byte pieces
// (E values a lane; !VEC: single values), a group of LPR lanes is a state of its own.  The keys and the values of a tile (U
// rows each per group) are all requested before the first is used.  It reads 8 x 32 heads of 4096 fp32 rows of 96 values
// in 119 us (6.8 TB/s) and of 256 in 321 (6.7), int8 rows of 96 in 41 (5.1); !VEC 8 x 32 x 4096 rows of 66 values in 196.
struct AttendArgs {
    PagedPool p;
    const float *q;
    float *out;
    float *part;    // [chunk of the launch][q_heads][d]: sums not yet divided (null: every sequence is one chunk)
    float2 *ml;     // [chunk of the launch][q_heads]: maximum and sum
    float *scores;  // accumulate: see scores_of
    int32_t *tickets;  // the last workgroup of a row joins its chunks (null: paged_join_kernel does)
    int n, q_heads, group, tiles_per_group, per_tile;
    int staged;  // words of LDS that page ids take before the scores that are kept there
    float scale;  // times log2 e
    int32_t slot[PAGED_BATCH], len[PAGED_BATCH], chunk[PAGED_BATCH];
    int32_t first[PAGED_BATCH + 1];          // first chunk of a sequence; INT_MAX behind the last sequence
    int64_t tokens_before[PAGED_BATCH];      // of the sequences before, each rounded up to a multiple of four
};
// The scores of one query head: [sequence][head][positions, rounded up to a multiple of four].
__device__ __forceinline__ float *scores_of(const AttendArgs &a, int i, int head) {
    return a.scores + a.tokens_before[i] * a.q_heads + (int64_t)head * ((a.len[i] + 3) & ~3);
}
// The sequence that chunk `b` belongs to: how many sequences end at or before it.
__device__ __forceinline__ int sequence_of(const AttendArgs &a, int b) {
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(a.first[lane + 1] <= b)) + __popcll(__ballot(a.first[lane + 65] <= b)));
}
template <bool Q8, bool VEC>
struct AttendRow {  // what a lane holds of a row, as it was loaded
    static constexpr int E = VEC && Q8 ? 16 : 4;
    int4 w;
    float s;
    __device__ __forceinline__ void load(const void *cache, const float *scales, int64_t row, int d, int l, bool ok) {
        w = make_int4(0, 0, 0, 0);
        s = 0.f;
        if (!ok) return;
        if (Q8) s = scales[row];
        if (VEC) {
            if (E * l < d) {
                const i32x4 x = stream(reinterpret_cast<const i32x4 *>((const char *)cache + row * d * (Q8 ? 1 : 4)) + l);
                w = make_int4(x[0], x[1], x[2], x[3]);
            }
        } else {
            const float *f = (const float *)cache + row * d;
            const signed char *c = (const signed char *)cache + row * d;
            if (l < d) w.x = Q8 ? (int)c[l] : __float_as_int(f[l]);
            if (l + 64 < d) w.y = Q8 ? (int)c[l + 64] : __float_as_int(f[l + 64]);
            if (l + 128 < d) w.z = Q8 ? (int)c[l + 128] : __float_as_int(f[l + 128]);
            if (l + 192 < d) w.w = Q8 ? (int)c[l + 192] : __float_as_int(f[l + 192]);
        }
    }
    __device__ __forceinline__ void widen(float (&x)[E]) const {  // int8: codes, without the scale
        const int ws[4] = {w.x, w.y, w.z, w.w};
        if (Q8 && VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int b = 0; b < 4; ++b) x[4 * j + b] = (float)(signed char)((ws[j] >> (8 * b)) & 0xff);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = Q8 ? (float)ws[j] : __int_as_float(ws[j]);
        }
    }
};
// Stores and loads that other dies see, past this one's L2.
__device__ __forceinline__ void put_through(float *p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float get_through(const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// The states that the wavefronts of a workgroup left in LDS ([head][wave][d] sums, [head][wave] maxima and sums) become the
// output, or the chunk's part of it.
template <int WAVES>
__device__ __forceinline__ void attend_merge(const AttendArgs &a, const float *so, const float *sm, const float *ss, int i, int b, int head0, int heads) {
    const int d = a.p.d;
    for (int j = threadIdx.x; j < heads * d; j += TPB) {
        const int g = j / d, c = j - g * d;
        float top = sm[g * WAVES];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sm[g * WAVES + w]);
        const float safe = top == -INFINITY ? 0.f : top;
        float o = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[g * WAVES + w] - safe);
            o += so[(g * WAVES + w) * d + c] * f;
            total += ss[g * WAVES + w] * f;
        }
        if (!a.part || (a.tickets && a.len[i] <= a.chunk[i])) {
            a.out[((int64_t)i * a.q_heads + head0 + g) * d + c] = a.len[i] > 0 ? o / total : 0.f;
        } else if (a.tickets) {
            put_through(&a.part[((int64_t)b * a.q_heads + head0 + g) * d + c], o);
            if (c == 0) {
                float *ml = reinterpret_cast<float *>(&a.ml[(int64_t)b * a.q_heads + head0 + g]);
                put_through(ml, top);
                put_through(ml + 1, total);
            }
        } else {
            a.part[((int64_t)b * a.q_heads + head0 + g) * d + c] = o;
            if (c == 0) a.ml[(int64_t)b * a.q_heads + head0 + g] = make_float2(top, total);
        }
    }
}
// Few rows of few chunks are joined by the workgroup that ends last.  Chunks of a row end on different dies, whose L2s do
// not see each other's lines: parts are stored past them (put_through), a workgroup takes its ticket when all its stores
// have arrived, and the one with the last ticket reads past its L2.  The chunks are added in order, whoever comes last.
// The ticket goes back to zero for the next launch.  The device takes as long as with the join's launch (48 rows of 577: 9.2
// us, 6.1 + 3.8 apart; 256 rows of 4096 int8 50.4, 46.6 + 4.6; of fp32 168, 162 + 5), but the host starts one less: where
// the rows do not fill the chip it is the host that a step waits for (a step with eviction over those 48 rows: 36.5 -> 31.8).
constexpr int LAST_CHUNKS = 8;
__device__ __forceinline__ void attend_last(const AttendArgs &a, int i, int head0, int heads) {
    __shared__ float share[16][LAST_CHUNKS], sums[16];
    __shared__ int taken;
    const int chunks = (a.len[i] + a.chunk[i] - 1) / a.chunk[i], d = a.p.d, tid = threadIdx.x;
    if (!a.tickets || chunks <= 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's stores have arrived
    __syncthreads();
    int32_t *ticket = a.tickets + i * (int)gridDim.y + (int)blockIdx.y;
    if (tid == 0) taken = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (taken != chunks - 1) return;
    if (tid == 0) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t first = a.first[i];
    if (tid < heads) {
        const float *ml = reinterpret_cast<const float *>(a.ml + first * a.q_heads + head0 + tid);
        float m[LAST_CHUNKS], s[LAST_CHUNKS], top = -INFINITY, total = 0.f;
#pragma unroll
        for (int c = 0; c < LAST_CHUNKS; ++c) {
            const int64_t at = 2 * (int64_t)min(c, chunks - 1) * a.q_heads;
            m[c] = get_through(ml + at);
            s[c] = get_through(ml + at + 1);
        }
#pragma unroll
        for (int c = 0; c < LAST_CHUNKS; ++c) top = fmaxf(top, m[c]);
        const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int c = 0; c < LAST_CHUNKS; ++c) {
            const float f = c < chunks ? __builtin_amdgcn_exp2f(m[c] - safe) : 0.f;
            share[tid][c] = f;
            if (c < chunks) total += s[c] * f;
        }
        sums[tid] = total;
    }
    __syncthreads();
    for (int j = tid; j < heads * d; j += TPB) {
        const int g = j / d;
        const float *part = a.part + (first * a.q_heads + head0) * d + j;
        float o = 0.f;
#pragma unroll 8
        for (int c = 0; c < chunks; ++c) o += get_through(part + (int64_t)c * a.q_heads * d) * share[g][c];
        a.out[((int64_t)i * a.q_heads + head0) * d + j] = o / sums[g];
    }
}
template <bool VEC, int E>
__device__ __forceinline__ int column_of(int l, int e) { return VEC ? l * E + e : l + 64 * e; }

template <bool Q8, bool VEC, int LPR, int U>
__global__ __launch_bounds__(TPB) void paged_attend_kernel(const AttendArgs a) {
    using Row = AttendRow<Q8, VEC>;
    constexpr int E = Row::E, RPP = 64 / LPR, TILE = RPP * U, WAVES = TPB / 64;
    extern __shared__ int32_t shared[];
    const PagedPool &p = a.p;
    const int d = p.d, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, sub = lane / LPR;
    const int b = blockIdx.x, i = sequence_of(a, b), head = blockIdx.y, h = head / a.group;
    const int t0 = (b - a.first[i]) * a.chunk[i], n = min(a.len[i] - t0, a.chunk[i]);
    // the chunk's pages
    const int p0 = t0 >> p.shift, pages = n > 0 ? ((t0 + n - 1) >> p.shift) - p0 + 1 : 0;
    for (int j = threadIdx.x; j < pages; j += TPB) shared[j] = p.table[a.slot[i] * p.max_pages + p0 + j];
    float qv[E], acc[E], m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = column_of<VEC, E>(l, e);
        acc[e] = 0.f;
        qv[e] = c < d ? a.q[((int64_t)i * a.q_heads + head) * d + c] : 0.f;
    }
    __syncthreads();
    for (int base = wave * TILE; base < n; base += WAVES * TILE) {
        Row k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = base + u * RPP + sub;
            const bool ok = t < n;
            const int64_t row = ok ? row_of(p, shared[((t0 + t) >> p.shift) - p0], h, (t0 + t) & (p.page - 1)) : 0;
            k[u].load(p.k, p.kscale, row, d, l, ok);
            v[u].load(p.v, p.vscale, row, d, l, ok);
        }
        float s[U], top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E], dot = 0.f;
            k[u].widen(x);
            const int t = base + u * RPP + sub;
#pragma unroll
            for (int e = 0; e < E; ++e) dot += qv[e] * x[e];
            dot = lanes_sum<LPR>(dot) * a.scale;
            if (Q8) dot *= k[u].s;
            s[u] = t < n ? dot : -INFINITY;
            if (a.scores && t < n && l == 0) scores_of(a, i, head)[t0 + t] = dot;
            top = fmaxf(top, s[u]);
        }
        const float safe = top == -INFINITY ? 0.f : top;  // nothing yet, or nothing but scores of -inf
        const float fade = __builtin_amdgcn_exp2f(m - safe);
        m = top;
        sum *= fade;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= fade;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = __builtin_amdgcn_exp2f(s[u] - safe);
            sum += s[u];
            if (Q8) s[u] *= v[u].s;
            float x[E];
            v[u].widen(x);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += s[u] * x[e];
        }
    }
    // the groups of a wavefront
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1) {
        const float mo = __shfl_xor(m, off, 64), so = __shfl_xor(sum, off, 64);
        const float top = fmaxf(m, mo), safe = top == -INFINITY ? 0.f : top;
        const float mine = __builtin_amdgcn_exp2f(m - safe), theirs = __builtin_amdgcn_exp2f(mo - safe);
        m = top;
        sum = sum * mine + so * theirs;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * mine + __shfl_xor(acc[e], off, 64) * theirs;
    }
    // the wavefronts of the workgroup
    __syncthreads();
    float *so = reinterpret_cast<float *>(shared), *sm = so + WAVES * d, *ss = sm + WAVES;
    if (sub == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = column_of<VEC, E>(l, e);
            if (c < d) so[wave * d + c] = acc[e];
        }
        if (l == 0) { sm[wave] = m; ss[wave] = sum; }
    }
    __syncthreads();
    attend_merge<WAVES>(a, so, sm, ss, i, b, head, 1);
    attend_last(a, i, head, 1);
}

// ---- the same on the matrix pipe -----------------------------------------------------------------------------------
// Up to 16 query heads of a key head make one side of a 16 x 16 tile, so a row of the cache is read once for all of
// them and the dot products cost no lane exchange.  Both products are taken transposed, which leaves a query head in
// every lane (head = lane % 16) from the scores to the output:
//   S^T = K Q^T   16 positions x 16 heads a tile; lane (head, quarter = lane / 16) gets positions 4 quarter .. + 3,
//   O^T += V^T P^T  contracts exactly those, so the probabilities go back into the matrix pipe from where they are.
// The order in which an MFMA contracts is free as long as both operands agree, which is what lets every load be 8 or 16
// contiguous bytes of a row: dims 16 j + 4 quarter .. + 3 for the fp32 keys, 4 (lane % 16) + 64 c .. + 3 for the values.
// fp32 rows: v_mfma_f32_16x16x4_f32 throughout.  int8 rows: the keys' codes are an operand as they lie in memory
// (v_mfma_i32_16x16x64_i8); a query is four 8-bit digits of its value over the largest of its head, 31 bits, half a
// unit of which is 2^-32 of that largest, and the integer sums are exact: beside a value ten thousand times theirs (in a dim
// where the keys are zero) the others' scores stay within the bound of fp32 sums, which three digits left.  The bytes of a
// biased integer are its digits, so the fourth costs no time (8 x 32 x 4096: 47.3 us with three, 47.4 with four).
// The values' codes are widened to bf16 (exact)
// and the probability, times the row's scale, is split into three bf16 parts that hold all of its 24 bits; products are
// exact and summed in fp32.  A wavefront keeps its tile's keys and values (and the next tile's keys) in registers.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float QUERY_UNITS = 127.0f * 16777216.0f;  // the largest query as an integer of four digits

// Where the rows of 16 positions lie.  The key row of a lane is position lane % 16, its value rows are 4 quarter + r.
// WIDE (pages of 16 positions and more): the 16 lie in one page, whose id is one scalar load from the table; rows are a
// scalar base and a 32-bit offset a lane.  Otherwise (pages of 4 and 8) every lane looks its rows up in the ids staged in
// LDS.  Positions behind the last are read as the last: every load is in bounds without a branch, and what must not count
// is cleared afterwards, in the last tile alone.
template <bool WIDE>
struct TileRows {
    int64_t key, value;  // WIDE: key is the first row, for all lanes
    int left;            // WIDE: positions behind the first that exist; else behind the first of the lane's four
    __device__ __forceinline__ void find(const PagedPool &p, const int32_t *table, const int32_t *staged, int p0, int h, int t, int last, int lane) {
        if (WIDE) {
            typedef const __attribute__((address_space(4))) int32_t *ConstInts;  // (nobody writes the table meanwhile)
            const int page = ((ConstInts)(uintptr_t)table)[t >> p.shift];
            key = value = row_of(p, page, h, t & (p.page - 1));
            left = last - t;
        } else {
            const int tk = min(t + (lane & 15), last), tv = min(t + 4 * (lane >> 4), last);
            key = row_of(p, staged[(tk >> p.shift) - p0], h, tk & (p.page - 1));
            value = row_of(p, staged[(tv >> p.shift) - p0], h, tv & (p.page - 1));
            left = last - tv;
        }
    }
    // addresses of this lane's rows in an array of `width` values a row, `column` values further on
    template <class E>
    __device__ __forceinline__ const E *key_at(const void *rows, int width, int column, int lane) const {
        const E *base = (const E *)rows + key * width;
        return WIDE ? base + (uint32_t)(min(lane & 15, left) * width + column) : base + column;
    }
    template <class E>
    __device__ __forceinline__ const E *value_at(const void *rows, int width, int column, int r, int lane) const {
        const E *base = (const E *)rows + value * width;
        return WIDE ? base + (uint32_t)(min(4 * (lane >> 4) + r, left) * width + column) : base + (uint32_t)(min(r, left) * width + column);
    }
    // the scales of the lane's four positions: on a multiple of four, in one page
    __device__ __forceinline__ const f32x4 *scales_at(const float *scales, int lane) const {
        return reinterpret_cast<const f32x4 *>(WIDE ? scales + key + (uint32_t)(4 * (lane >> 4)) : scales + (value & ~(int64_t)3));
    }
};

// The running state of a wavefront: maximum and sum of a head (equal in its four lanes; the sum is a lane's own part),
// outputs of `N` tiles of 16 dims.
template <int N>
struct TileState {
    float m, sum;
    f32x4 o[N];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // scores of 16 T positions become probabilities under the new maximum
    template <int T>
    __device__ __forceinline__ void take(f32x4 (&s)[T]) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < T; ++t) top = fmaxf(top, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
        float a, b;
        swap16(top, a, b);
        top = fmaxf(a, b);
        swap32(top, a, b);
        top = fmaxf(fmaxf(a, b), m);
        const float safe = top == -INFINITY ? 0.f : top;
        if (__any(top != m)) {  // (after a few tiles the maximum seldom moves)
            const float fade = __builtin_amdgcn_exp2f(m - safe);
            m = top;
            sum *= fade;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] *= fade;
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - safe);
                sum += s[t][r];
            }
    }
};
// The wavefronts' states of one workgroup come together and leave: dim_of(tile, row) is the dim of row `row` of tile i.
template <int N, class F>
__device__ __forceinline__ void tile_finish(const AttendArgs &a, TileState<N> &st, float *lds, int i, int b, int head0, int heads, F dim_of) {
    constexpr int WAVES = TPB / 64;
    const int d = a.p.d, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane & 15;
    float x, y;
    swap16(st.sum, x, y);
    st.sum = x + y;
    swap32(st.sum, x, y);
    st.sum = x + y;
    __syncthreads();  // (the pages' ids are read no more)
    float *sm = lds, *ss = sm + 16 * WAVES, *so = ss + 16 * WAVES;  // so: [head][wave][d]
    if (lane < 16) { sm[g * WAVES + wave] = st.m; ss[g * WAVES + wave] = st.sum; }
    if (g < heads) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = dim_of(j, 4 * (lane >> 4) + r);
                if (c < d) so[(g * WAVES + wave) * d + c] = st.o[j][r];
            }
    }
    __syncthreads();
    attend_merge<WAVES>(a, so, sm, ss, i, b, head0, heads);
    attend_last(a, i, head0, heads);
}
// What both kernels begin with.
struct TileWork {
    int i, h, head0, heads, t0, n, p0, chunk;
    const int32_t *table;
};
template <bool WIDE>
__device__ __forceinline__ TileWork tile_work(const AttendArgs &a, int32_t *staged) {
    const PagedPool &p = a.p;
    TileWork w;
    w.i = sequence_of(a, blockIdx.x);
    w.h = blockIdx.y / a.tiles_per_group;
    const int g0 = (blockIdx.y % a.tiles_per_group) * a.per_tile;
    w.t0 = (blockIdx.x - a.first[w.i]) * a.chunk[w.i];
    w.chunk = a.chunk[w.i];
    w.n = min(a.len[w.i] - w.t0, w.chunk);
    w.head0 = w.h * a.group + g0;
    w.heads = min(a.per_tile, a.group - g0);
    w.p0 = w.t0 >> p.shift;
    w.table = p.table + a.slot[w.i] * p.max_pages;
    if (!WIDE) {
        const int count = w.n > 0 ? ((w.t0 + w.n - 1) >> p.shift) - w.p0 + 1 : 0;
        for (int j = threadIdx.x; j < count; j += TPB) staged[j] = w.table[w.p0 + j];
        __syncthreads();
    }
    return w;
}
// accumulate: a chunk's scores are kept in LDS, [head][positions + 4] (the odd 16 bytes spread a wavefront's four quarters
// over the banks), and leave at the end in whole lines, past the caches.  On 131072 positions of 32 heads (17 MB among 1.1
// GB of reads) they cost 14 us so, 20 through the caches, and 34 written tile by tile, 64 bytes a head.
template <int T>
__device__ __forceinline__ void tile_scores_keep(float *scores, const TileWork &w, const f32x4 (&s)[T], int base, int lane) {
    if ((lane & 15) >= w.heads) return;
    float *row = scores + (lane & 15) * (w.chunk + 4);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const int at = base + 16 * t + 4 * (lane >> 4);
        if (at < w.n) *reinterpret_cast<f32x4 *>(row + at) = s[t];
    }
}
__device__ __forceinline__ void tile_scores_out(const AttendArgs &a, const TileWork &w, const float *scores) {
    __syncthreads();
    for (int g = 0; g < w.heads; ++g) {
        float *out = scores_of(a, w.i, w.head0 + g) + w.t0;  // (a head's row begins on a multiple of four and is as long as one)
        for (int at = 4 * (int)threadIdx.x; at < w.n; at += 4 * TPB)
            __builtin_nontemporal_store(*reinterpret_cast<const f32x4 *>(scores + g * (w.chunk + 4) + at), reinterpret_cast<f32x4 *>(out + at));
    }
}

// NC blocks of 64 dims (d a multiple of 4; EVEN: d = 64 NC), 16 * T positions a turn of a wavefront.  Keys of the next turn
// are asked for when the scores are done with this turn's, values when the outputs are: every wavefront has a tile's keys
// or values on the way at any time without a second set of registers.  The queries stay in LDS (8 reads a turn for 32
// registers).  Bound by bandwidth from one query head a key head to eight: 8 x 32 heads of 4096 rows of 128 values 159 us
// (6.75 TB/s), 192 values 242, 256 values 328 (6.5; 389 with clamped columns).
template <int NC, int T, bool EVEN, bool WIDE>
__global__ __launch_bounds__(TPB, NC <= 2 ? 3 : 1) void paged_attend_tiles_kernel(const AttendArgs a) {
    constexpr int WAVES = TPB / 64, TILE = 16 * T;
    extern __shared__ int32_t shared[];
    __shared__ f32x4 qs[NC * 4][64];  // [16 dims][lane]
    const PagedPool &p = a.p;
    const int d = EVEN ? 64 * NC : p.d, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, quarter = lane >> 4;
    const TileWork w = tile_work<WIDE>(a, shared);
    const int last = w.t0 + w.n - 1;
    float *scores = reinterpret_cast<float *>(shared) + (WIDE ? 0 : a.staged);
    TileState<NC * 4> st;
    st.clear();
    f32x4 k[T][NC * 4], v[T][NC][4];
    TileRows<WIDE> rows[T];
    auto load_keys = [&](int base) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            rows[t].find(p, w.table, shared, w.p0, w.h, min(w.t0 + base + 16 * t, last & ~15), last, lane);
#pragma unroll
            for (int j = 0; j < NC * 4; ++j) {
                const int c = 16 * j + 4 * quarter;
                k[t][j] = stream(reinterpret_cast<const f32x4 *>(rows[t].template key_at<float>(p.k, d, EVEN || c < d ? c : 0, lane)));
                if (!EVEN && c >= d) k[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    };
    auto load_values = [&](int base) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int col = 64 * c + 4 * m16;
                    v[t][c][r] = stream(reinterpret_cast<const f32x4 *>(rows[t].template value_at<float>(p.v, d, EVEN || col < d ? col : 0, r, lane)));
                }
    };
    int base = wave * TILE;
    if (base < w.n) {
        load_keys(base);
        load_values(base);
    }
    for (int j = wave; j < NC * 4; j += WAVES) {
        const int c = 16 * j + 4 * quarter;
        qs[j][lane] = m16 < w.heads && c < d ? *reinterpret_cast<const f32x4 *>(a.q + ((int64_t)w.i * a.q_heads + w.head0 + m16) * d + c) * a.scale
                                             : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    for (; base < w.n; base += WAVES * TILE) {
        const int next = base + WAVES * TILE;
        f32x4 s[T], s2[T];  // (two sums: half the roundings)
#pragma unroll
        for (int t = 0; t < T; ++t) s[t] = s2[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NC * 4; ++j) {
            const f32x4 q = qs[j][lane];
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f32x4 &to = j & 1 ? s2[t] : s[t];
                    to = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][j][e], q[e], to, 0, 0, 0);
                }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) s[t] += s2[t];
        if (next < w.n) load_keys(next);
        if (a.scores) tile_scores_keep<T>(scores, w, s, base, lane);
        if (base + TILE > w.n) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (base + 16 * t + 4 * quarter + r >= w.n) {
                        s[t][r] = -INFINITY;
#pragma unroll
                        for (int c = 0; c < NC; ++c) v[t][c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
        }
        st.template take<T>(s);
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[4 * c + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][c][r][e], s[t][r], st.o[4 * c + e], 0, 0, 0);
        if (next < w.n) load_values(next);
    }
    if (a.scores) tile_scores_out(a, w, scores);
    tile_finish(a, st, reinterpret_cast<float *>(shared), w.i, blockIdx.x, w.head0, w.heads, [](int j, int row) { return 64 * (j >> 2) + 4 * row + (j & 3); });
}

// int8.  ND blocks of 64 dims for the keys; a lane widens NE dims of the values, NE * (lane % 16) .. + NE - 1 (d a multiple
// of 16, EVEN: d = 64 ND = 16 NE).  32 positions a turn: one step of the bf16 product.
template <int ND, int NE, bool EVEN, bool WIDE>
__global__ __launch_bounds__(TPB, NE <= 8 ? 3 : 1) void paged_attend_tiles_i8_kernel(const AttendArgs a) {
    constexpr int WAVES = TPB / 64, T = 2, TILE = 16 * T, VW = NE / 4;
    typedef int32_t Word __attribute__((ext_vector_type(VW)));
    extern __shared__ int32_t shared[];
    __shared__ i32x4 digits[4][ND][64];  // [digit][64 dims][lane]
    __shared__ float units_of[16];
    const PagedPool &p = a.p;
    const int d = EVEN ? 64 * ND : p.d, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, quarter = lane >> 4;
    const TileWork w = tile_work<WIDE>(a, shared);
    const int last = w.t0 + w.n - 1;
    float *scores = reinterpret_cast<float *>(shared) + (WIDE ? 0 : a.staged);
    TileState<NE> st;
    st.clear();
    i32x4 k[T][ND];
    f32x4 ks[T], vs[T];
    Word v[T][4];
    TileRows<WIDE> rows[T];
    auto load_keys = [&](int base) {  // and their scales
#pragma unroll
        for (int t = 0; t < T; ++t) {
            rows[t].find(p, w.table, shared, w.p0, w.h, min(w.t0 + base + 16 * t, last & ~15), last, lane);
#pragma unroll
            for (int j = 0; j < ND; ++j) {  // (beyond d the digits are zeros)
                const int c = 64 * j + 16 * quarter;
                k[t][j] = stream(reinterpret_cast<const i32x4 *>(rows[t].template key_at<signed char>(p.k, d, EVEN || c < d ? c : 0, lane)));
            }
            ks[t] = *rows[t].scales_at(p.kscale, lane);
        }
    };
    auto load_values = [&](int base) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[t][r] = stream(reinterpret_cast<const Word *>(rows[t].template value_at<signed char>(p.v, d, EVEN || NE * m16 < d ? NE * m16 : 0, r, lane)));
            vs[t] = *rows[t].scales_at(p.vscale, lane);
        }
    };
    int base = wave * TILE;
    if (base < w.n) {
        load_keys(base);
        load_values(base);
    }
    // the query's digits: dims 64 j + 16 quarter .. + 15 of head m16, and what one unit of them stands for
    if (wave == 0) {
        const bool mine = m16 < w.heads;
        const float *qr = a.q + ((int64_t)w.i * a.q_heads + w.head0 + (mine ? m16 : 0)) * d + 16 * quarter;
        f32x4 x[ND][4];
        float top = 0.f, check = 0.f;
#pragma unroll
        for (int j = 0; j < ND; ++j) {
            const bool ok = mine && (EVEN || 64 * j + 16 * quarter < d);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                x[j][y] = EVEN || ok ? *reinterpret_cast<const f32x4 *>(qr + 64 * j + 4 * y) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[j][y][e] = ok ? x[j][y][e] : 0.f;
                    top = fmaxf(top, fabsf(x[j][y][e]));
                    check += x[j][y][e] * 0.f;  // NaN where a value is infinite or NaN
                }
            }
        }
        float u, v;
        swap16(top, u, v);
        top = fmaxf(u, v);
        swap32(top, u, v);
        top = fmaxf(u, v);
        swap16(check, u, v);
        check = u + v;
        swap32(check, u, v);
        check = u + v;
        top = fmaxf(top, 1e-29f);  // (below, `units` would be infinite)
        const float units = QUERY_UNITS / top;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int whole = (int)rintf((check == 0.f ? x[j][y][e] : 0.f) * units);
                    w[e] = ((uint32_t)whole + 0x808080u) ^ 0x808080u;  // its bytes are digits from -128 to 127 that make it up
                }
                const uint32_t low01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), high01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
                const uint32_t low23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), high23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
                const uint32_t pack[4] = {__builtin_amdgcn_perm(high23, high01, 0x07060302), __builtin_amdgcn_perm(high23, high01, 0x05040100),
                                          __builtin_amdgcn_perm(low23, low01, 0x07060302), __builtin_amdgcn_perm(low23, low01, 0x05040100)};
#pragma unroll
                for (int z = 0; z < 4; ++z) reinterpret_cast<uint32_t *>(&digits[z][j][lane])[y] = pack[z];
            }
        if (lane < 16) units_of[lane] = (top * (256.0f / QUERY_UNITS) + check) * a.scale;
    }
    __syncthreads();
    const float unit = units_of[m16];
    for (; base < w.n; base += WAVES * TILE) {
        const int next = base + WAVES * TILE;
        f32x4 s[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            i32x4 x[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                x[y] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < ND; ++j) x[y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][j], digits[y][j][lane], x[y], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[t][r] = ((float)(x[0][r] * 256 + x[1][r]) * 256.0f + (float)(x[2][r] * 256 + x[3][r]) * 0x1p-8f) * (ks[t][r] * unit);
        }
        if (next < w.n) load_keys(next);
        if (a.scores) tile_scores_keep<T>(scores, w, s, base, lane);
        if (base + TILE > w.n) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (base + 16 * t + 4 * quarter + r >= w.n) {
                        s[t][r] = -INFINITY;
                        vs[t][r] = 0.f;
                    }
        }
        st.template take<T>(s);
        // (an opaque use: without it the compiler carries the codes over the loop's edge byte by byte, a register each)
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < VW; ++x) {
                    int32_t word = v[t][r][x];
                    asm volatile("" : "+v"(word));
                    v[t][r][x] = word;
                }
        // p times the row's scale in three parts: the upper 8 bits of the significand, the next 8, the rest
        i32x4 part[3];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            uint32_t up[3][2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int t = x >> 1, r = 2 * (x & 1) + y;
                const float f = s[t][r] * vs[t][r];
                up[0][y] = __float_as_uint(f) & 0xffff0000u;
                const float rest = f - __uint_as_float(up[0][y]);
                up[1][y] = __float_as_uint(rest) & 0xffff0000u;
                up[2][y] = __float_as_uint(rest - __uint_as_float(up[1][y]));
            }
#pragma unroll
            for (int y = 0; y < 3; ++y) part[y][x] = (int)__builtin_amdgcn_perm(up[y][1], up[y][0], 0x07060302);
        }
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            i32x4 col;  // dim NE m16 + e of the eight rows
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int t = x >> 1, r = 2 * (x & 1), sh = 8 * (e & 3);
                const float lo = (float)(signed char)(v[t][r][e >> 2] >> sh), hi = (float)(signed char)(v[t][r + 1][e >> 2] >> sh);
                col[x] = (int)__builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
            }
#pragma unroll
            for (int y = 2; y >= 0; --y)
                st.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, col), __builtin_bit_cast(bf16x8, part[y]), st.o[e], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (next < w.n) load_values(next);
    }
    if (a.scores) tile_scores_out(a, w, scores);
    tile_finish(a, st, reinterpret_cast<float *>(shared), w.i, blockIdx.x, w.head0, w.heads, [](int j, int row) { return NE * row + j; });
}

// What follows the chunks, in one launch.  The first `joins` workgroups join them, each 32 values of an output row (few
// rows of many chunks are the case that takes long): every chunk's share of the row's sum first (one thread a chunk), then
// W values a thread and the chunks dealt over the threads that share a column, added up in a fixed order.  accumulate: the
// others add the probabilities of 1024 positions of one sequence and key head, summed over its query heads, to their
// weights, and work the row's maximum and sum out of the chunks' again (some hundred values): waiting for the joins that
// have them would be a launch of its own, 3.5 us.
constexpr int JOIN_CHUNKS = 1024;
__device__ __forceinline__ float2 join_stats(const AttendArgs &a, int first, int chunks, int head, int lane) {  // by one wavefront
    float top = -INFINITY, total = 0.f;
    for (int c = lane; c < chunks; c += 64) {
        const float2 s = a.ml[(int64_t)(first + c) * a.q_heads + head];
        const float next = fmaxf(top, s.x), safe = next == -INFINITY ? 0.f : next;
        total = total * __builtin_amdgcn_exp2f(top - safe) + s.y * __builtin_amdgcn_exp2f(s.x - safe);
        top = next;
    }
    const float all = lanes_max<64>(top), safe = all == -INFINITY ? 0.f : all;
    return make_float2(safe, lanes_sum<64>(total * __builtin_amdgcn_exp2f(top - safe)));
}
template <int W>
__device__ __forceinline__ void attend_join(const AttendArgs &a, float *share, float (*sums)[W], int row, int block) {
    const int tid = threadIdx.x, lane = tid & 63;
    constexpr int COLS = 32 / W, GROUPS = TPB / COLS;
    const int i = row / a.q_heads, head = row - i * a.q_heads;
    const int first = a.first[i], chunks = (a.len[i] + a.chunk[i] - 1) / a.chunk[i];
    const float2 whole = join_stats(a, first, chunks, head, lane);  // (every wavefront for itself: the same bits)
    const int column = 32 * block + W * (tid % COLS), group = tid / COLS;
    const bool live = column < a.p.d;
    float o[W];
#pragma unroll
    for (int e = 0; e < W; ++e) o[e] = 0.f;
    for (int c0 = 0; c0 < chunks; c0 += JOIN_CHUNKS) {
        const int some = min(chunks - c0, JOIN_CHUNKS);
        __syncthreads();
        for (int c = tid; c < some; c += TPB) share[c] = __builtin_amdgcn_exp2f(a.ml[(int64_t)(first + c0 + c) * a.q_heads + head].x - whole.x);
        __syncthreads();
        if (live) {
            const float *part = a.part + ((int64_t)(first + c0) * a.q_heads + head) * a.p.d + column;
#pragma unroll 4
            for (int c = group; c < some; c += GROUPS) {
                float x[W];
                __builtin_memcpy(x, __builtin_assume_aligned(part + (int64_t)c * a.q_heads * a.p.d, 4 * W), 4 * W);
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] += x[e] * share[c];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) sums[tid][e] = o[e];
    __syncthreads();
    if (tid < 32 && 32 * block + tid < a.p.d) {
        float sum = 0.f;
        for (int g = 0; g < GROUPS; ++g) sum += sums[g * COLS + tid / W][tid % W];
        a.out[(int64_t)row * a.p.d + 32 * block + tid] = chunks > 0 ? sum / whole.y : 0.f;
    }
}
__device__ __forceinline__ void attend_weights(const AttendArgs &a, float2 *stats, int row, int block) {
    constexpr int WAVES = TPB / 64;
    const int i = row / a.p.heads, h = row - i * a.p.heads, len = a.len[i], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (block * 4 * TPB >= len) return;  // (the whole workgroup)
    const int t = 4 * (block * TPB + (int)threadIdx.x), first = a.first[i], chunks = (len + a.chunk[i] - 1) / a.chunk[i];
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int g0 = 0; g0 < a.group; g0 += WAVES) {
        const int some = min(WAVES, a.group - g0);
        __syncthreads();
        if (wave < some) {
            const float2 s = join_stats(a, first, chunks, h * a.group + g0 + wave, lane);
            if (lane == 0) stats[wave] = make_float2(s.x, 1.0f / s.y);
        }
        f32x4 x[WAVES];
#pragma unroll
        for (int g = 0; g < WAVES; ++g)
            if (t < len && g < some) x[g] = *reinterpret_cast<const f32x4 *>(scores_of(a, i, h * a.group + g0 + g) + t);
        __syncthreads();
#pragma unroll
        for (int g = 0; g < WAVES; ++g)
            if (t < len && g < some) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] += __builtin_amdgcn_exp2f(x[g][e] - stats[g].x) * stats[g].y;
            }
    }
    float *weight = a.p.weight + ((int64_t)a.slot[i] * a.p.heads + h) * a.p.max_len + t;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (t + e < len) weight[e] += w[e];
}
template <int W>
__global__ __launch_bounds__(TPB) void paged_join_kernel(const AttendArgs a, int joins, int tiles) {
    __shared__ float share[JOIN_CHUNKS], sums[TPB][W];
    const int b = blockIdx.x, blocks = (a.p.d + 31) / 32;
    if (b < joins) attend_join<W>(a, share, sums, b / blocks, b % blocks);
    else attend_weights(a, reinterpret_cast<float2 *>(share), (b - joins) / tiles, (b - joins) % tiles);
}

template <bool Q8, bool VEC, int LPR, int U>
void launch_attend(const AttendArgs &a, int chunks, int widest) {
    const int pages = widest / a.p.page + 2, merge = (TPB / 64) * (a.p.d + 2);
    const size_t lds = (size_t)(pages > merge ? pages : merge) * 4;
    MNI_KERNEL_LAUNCH((paged_attend_kernel<Q8, VEC, LPR, U>), dim3((unsigned)chunks, (unsigned)a.q_heads), dim3(TPB), lds, ctx().stream, a);
}
template <class K>
void launch_tiles(K kernel, AttendArgs &a, int chunks, int widest) {
    const int heads = a.group < a.per_tile ? a.group : a.per_tile, merge = (TPB / 64) * (32 + heads * a.p.d);
    a.staged = a.p.page >= 16 ? 0 : (widest / a.p.page + 2 + 3) & ~3;
    const int during = a.staged + (a.scores ? heads * (widest + 4) : 0);
    const size_t lds = (size_t)(during > merge ? during : merge) * 4;
    MNI_KERNEL_LAUNCH(kernel, dim3((unsigned)chunks, (unsigned)(a.p.heads * a.tiles_per_group)), dim3(TPB), lds, ctx().stream, a);
}

}  // namespace

// The positions of a chunk: as few as still leave every workgroup of the launch resident at once (they then start and
// end together and no CU waits for a last round), never under ATTEND_LEAST (a workgroup's start and end are worth some
// hundred positions).  Where even one chunk per row is more than the chip holds, a quarter of an even share.
constexpr int ATTEND_STEP = 64, ATTEND_LEAST = 128, ATTEND_MOST = 8192;
static int64_t attend_chunk(const PagedSeqs &s, int64_t rows, int64_t tokens, int64_t resident, int64_t most) {
    auto workgroups = [&](int64_t chunk) {
        int64_t n = 0;
        for (int i = 0; i < s.n; ++i) n += s.len[i] > chunk ? (s.len[i] + chunk - 1) / chunk : 1;
        return n * rows;
    };
    int64_t lo = 1, hi = most / ATTEND_STEP;
    if (workgroups(hi * ATTEND_STEP) > resident) {
        int64_t chunk = tokens * rows / (4 * resident) / ATTEND_STEP * ATTEND_STEP;
        chunk = chunk < 4 * ATTEND_LEAST ? 4 * ATTEND_LEAST : chunk;
        return chunk > most ? most : chunk;
    }
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (workgroups(mid * ATTEND_STEP) <= resident) hi = mid;
        else lo = mid + 1;
    }
    const int64_t chunk = lo * ATTEND_STEP;
    return chunk < ATTEND_LEAST ? ATTEND_LEAST : chunk;
}

int k_paged_attend(const PagedPool &p, const PagedSeqs &s, const float *q, float *out, int q_heads, float scale, bool accumulate) {
    if (s.n <= 0) return MNI_OK;
    AttendArgs a;
    a.p = p;
    a.q = q;
    a.out = out;
    a.part = nullptr;
    a.ml = nullptr;
    a.scores = nullptr;
    a.tickets = nullptr;
    a.n = s.n;
    a.q_heads = q_heads;
    a.group = q_heads / p.heads;
    a.scale = scale * LOG2E;
    int64_t tokens = 0, longest = 0;
    for (int i = 0; i < s.n; ++i) {
        tokens += s.len[i];
        if (s.len[i] > longest) longest = s.len[i];
    }
    const int64_t cus = ctx().compute_units > 0 ? ctx().compute_units : 256;
    // 16-byte pieces of a row: both forms want them.  The matrix pipe's also wants pages of at least four positions.  Query
    // heads that share a key head are its gain (us, 8 sequences of 4096, 32 query heads, fp32 rows of 128: 16 key heads 83,
    // vector form 110; 8: 45 and 90; int8 18 and 41).  Without them it still is as quick where its loads need no clamping and its rows no
    // lookups (dims in 64s and pages from 16 on: fp32 159 and 161, 192 dims 242 and 238, 256 328 and 319; int8 47 and 46,
    // 256 dims 85 and 88), else slower (96 dims 178 and 119; pages of 8, 128 dims: 198 and 164; int8, 96 dims: 45 and 41);
    // fp32 rows of other dims than 64s even for two heads (96: 87 and 81, 32: 40 and 29; three heads of 96: 50 and 57).
    // Where the rows do not fill the chip the start and end of a workgroup count, and the vector form's are shorter for
    // fp32 (57 rows of 12 heads: 5.4 and 4.5; 4 x 577: 6.7 and 6.1), for int8 not (4 x 2047, 12 heads: 7.2 and 8.6).
    const bool vec = p.d % (p.quantized ? 16 : 4) == 0 && ((uintptr_t)q & 15) == 0;
    const bool few = tokens * p.heads < cus * 3 * ATTEND_LEAST;
    const bool tiles = vec && p.page >= 4 && (a.group > (p.quantized || p.d % 64 == 0 ? 1 : 2) || (p.d % 64 == 0 && p.page >= 16 && (p.quantized || !few)));
    a.per_tile = !tiles ? 1 : p.d <= 128 ? 16 : 8;  // (the merge of 16 heads of 256 dims would not fit 64 KB of LDS)
    a.tiles_per_group = (a.group + a.per_tile - 1) / a.per_tile;
    const int64_t rows = (int64_t)p.heads * a.tiles_per_group;
    // as many workgroups as the registers let a CU hold; scores that are kept in LDS shall take 44 KB of it at most
    const int64_t kept = 11264 / (a.group < a.per_tile ? a.group : a.per_tile) / ATTEND_STEP * ATTEND_STEP;
    const int64_t target = attend_chunk(s, rows, tokens, cus * (p.d <= 128 ? 3 : tiles ? 1 : 2), accumulate && tiles && kept < ATTEND_MOST ? kept : ATTEND_MOST);
    int chunks = 0;
    int64_t before = 0, widest = 0;
    int64_t most = 0;  // chunks of a row
    for (int i = 0; i < PAGED_BATCH; ++i) {
        const int64_t len = i < s.n ? s.len[i] : 0;
        a.slot[i] = i < s.n ? s.slot[i] : 0;
        a.len[i] = (int32_t)len;
        a.first[i] = i < s.n ? chunks : INT_MAX;
        a.tokens_before[i] = before;
        const int64_t c = len > target ? (len + target - 1) / target : 1;  // (an empty sequence: one that writes zeros)
        int64_t chunk = (len + c - 1) / c;
        chunk = chunk > 0 ? (chunk + ATTEND_STEP - 1) / ATTEND_STEP * ATTEND_STEP : ATTEND_STEP;
        a.chunk[i] = (int32_t)chunk;
        if (i < s.n) {
            const int64_t used = len > 0 ? (len + chunk - 1) / chunk : 1;
            if (used > most) most = used;
            chunks += (int)used;
            before += (len + 3) & ~(int64_t)3;
            if (chunk > widest) widest = chunk;
        }
    }
    a.first[PAGED_BATCH] = INT_MAX;
    const int64_t joins = (int64_t)s.n * q_heads * ((p.d + 31) / 32), strips = (longest + 4 * TPB - 1) / (4 * TPB);
    const int64_t tail = joins + (accumulate ? s.n * p.heads * strips : 0);  // workgroups behind the chunks': see paged_join_kernel
    if (s.n > 1 && (chunks > most_blocks(TPB) || tail > most_blocks(TPB))) {  // (one sequence alone outgrows the memory before a grid)
        for (int from : {0, s.n / 2}) {
            PagedSeqs half;
            half.n = from ? s.n - from : s.n / 2;
            for (int i = 0; i < half.n; ++i) { half.slot[i] = s.slot[from + i]; half.len[i] = s.len[from + i]; }
            const int64_t at = (int64_t)from * q_heads * p.d;
            MNI_TRY(k_paged_attend(p, half, q + at, out + at, q_heads, scale, accumulate));
        }
        return MNI_OK;
    }
    void *part = nullptr, *ml = nullptr, *scores = nullptr;
    int rc = MNI_OK;
    const bool last = few && !accumulate && most <= LAST_CHUNKS && s.n * rows <= PAGED_TICKETS;
    if (most > 1 || accumulate) {
        if (last) a.tickets = p.tickets;
        rc = dev_alloc(&part, (size_t)chunks * q_heads * p.d * sizeof(float));
        if (rc == MNI_OK) rc = dev_alloc(&ml, (size_t)chunks * q_heads * sizeof(float2));
        if (rc == MNI_OK && accumulate) rc = dev_alloc(&scores, (size_t)(before > 0 ? before : 1) * q_heads * sizeof(float));
        a.part = (float *)part;
        a.ml = (float2 *)ml;
        a.scores = (float *)scores;
    }
    if (rc == MNI_OK) {
        const int w = (int)widest;
        if (tiles && p.quantized && p.page >= 16) {
            if (p.d == 64) launch_tiles(paged_attend_tiles_i8_kernel<1, 4, true, true>, a, chunks, w);
            else if (p.d < 64) launch_tiles(paged_attend_tiles_i8_kernel<1, 4, false, true>, a, chunks, w);
            else if (p.d == 128) launch_tiles(paged_attend_tiles_i8_kernel<2, 8, true, true>, a, chunks, w);
            else if (p.d < 128) launch_tiles(paged_attend_tiles_i8_kernel<2, 8, false, true>, a, chunks, w);
            else launch_tiles(paged_attend_tiles_i8_kernel<4, 16, false, true>, a, chunks, w);
        } else if (tiles && p.quantized) {
            if (p.d <= 64) launch_tiles(paged_attend_tiles_i8_kernel<1, 4, false, false>, a, chunks, w);
            else if (p.d <= 128) launch_tiles(paged_attend_tiles_i8_kernel<2, 8, false, false>, a, chunks, w);
            else launch_tiles(paged_attend_tiles_i8_kernel<4, 16, false, false>, a, chunks, w);
        } else if (tiles && p.page >= 16) {
            if (p.d == 64) launch_tiles(paged_attend_tiles_kernel<1, 2, true, true>, a, chunks, w);
            else if (p.d < 64) launch_tiles(paged_attend_tiles_kernel<1, 2, false, true>, a, chunks, w);
            else if (p.d == 128) launch_tiles(paged_attend_tiles_kernel<2, 1, true, true>, a, chunks, w);
            else if (p.d < 128) launch_tiles(paged_attend_tiles_kernel<2, 1, false, true>, a, chunks, w);
            else if (p.d == 192) launch_tiles(paged_attend_tiles_kernel<3, 1, true, true>, a, chunks, w);
            else if (p.d < 192) launch_tiles(paged_attend_tiles_kernel<3, 1, false, true>, a, chunks, w);
            else if (p.d == 256) launch_tiles(paged_attend_tiles_kernel<4, 1, true, true>, a, chunks, w);
            else launch_tiles(paged_attend_tiles_kernel<4, 1, false, true>, a, chunks, w);
        } else if (tiles) {
            if (p.d <= 64) launch_tiles(paged_attend_tiles_kernel<1, 2, false, false>, a, chunks, w);
            else if (p.d <= 128) launch_tiles(paged_attend_tiles_kernel<2, 1, false, false>, a, chunks, w);
            else launch_tiles(paged_attend_tiles_kernel<4, 1, false, false>, a, chunks, w);
        } else if (!vec) {
            if (p.quantized) launch_attend<true, false, 64, 4>(a, chunks, w);
            else launch_attend<false, false, 64, 4>(a, chunks, w);
        } else if (p.quantized) {
            if (p.d <= 64) launch_attend<true, true, 4, 4>(a, chunks, w);
            else if (p.d <= 128) launch_attend<true, true, 8, 4>(a, chunks, w);
            else launch_attend<true, true, 16, 8>(a, chunks, w);
        } else {
            if (p.d <= 32) launch_attend<false, true, 8, 4>(a, chunks, w);
            else if (p.d <= 64) launch_attend<false, true, 16, 4>(a, chunks, w);
            else if (p.d <= 128) launch_attend<false, true, 32, 4>(a, chunks, w);
            else launch_attend<false, true, 64, 8>(a, chunks, w);
        }
        rc = check_launch("paged_attend");
    }
    if (rc == MNI_OK && a.part && !last) {
        const dim3 grid((unsigned)tail);
        if (p.d % 4 == 0) MNI_KERNEL_LAUNCH(paged_join_kernel<4>, grid, dim3(TPB), 0, ctx().stream, a, (int)joins, (int)strips);
        else MNI_KERNEL_LAUNCH(paged_join_kernel<1>, grid, dim3(TPB), 0, ctx().stream, a, (int)joins, (int)strips);
        rc = check_launch("paged_join");
    }
    if (part) dev_free(part);
    if (ml) dev_free(ml);
    if (scores) dev_free(scores);
    return rc;
}

}  // namespace mni
