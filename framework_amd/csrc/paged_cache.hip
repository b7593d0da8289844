// Kernels of the paged key-value cache (mni_paged_cache_*): append, attention of one new token per sequence over its
// pages, eviction by accumulated weight.  All of them are bound by memory: a decoding step reads every key and value
// row it attends to once, which is all it has to do.
#include <limits.h>

#include <vector>

#include "lanes.h"
#include "paged_cache.h"

namespace mni {
namespace {

constexpr int TPB = 256;
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int64_t row_of(const PagedPool &p, int page, int head, int slot) {
    return ((int64_t)page * p.heads + head) * p.page + slot;
}

// ---- table entries, page copies, forks -----------------------------------------------------------------------------
__global__ __launch_bounds__(TPB) void paged_table_kernel(int32_t *__restrict__ table, const PagedTableWrite w) {
    for (int i = threadIdx.x; i < w.n; i += TPB) table[w.at[i]] = w.page[i];
}
// blockIdx.x: the copy, blockIdx.y: keys, values, key scales, value scales.  A page is one contiguous block.
__global__ __launch_bounds__(TPB) void paged_copy_kernel(const PagedPool p, const PagedCopies c) {
    const int what = blockIdx.y;
    const int64_t rows = (int64_t)p.heads * p.page, unit = what >= 2 || !p.quantized ? 4 : 1;
    const int64_t bytes = rows * (what >= 2 ? 1 : p.d) * unit;
    char *base = (char *)(what == 0 ? p.k : what == 1 ? p.v : what == 2 ? (void *)p.kscale : (void *)p.vscale);
    const char *src = base + c.from[blockIdx.x] * bytes;
    char *dst = base + c.to[blockIdx.x] * bytes;
    if (bytes % 16 == 0) {
        for (int64_t i = threadIdx.x; i < bytes / 16; i += TPB) reinterpret_cast<int4 *>(dst)[i] = reinterpret_cast<const int4 *>(src)[i];
    } else {
        for (int64_t i = threadIdx.x; i < bytes; i += TPB) dst[i] = src[i];
    }
    if (what == 0 && threadIdx.x == 0) p.table[c.at[blockIdx.x]] = c.to[blockIdx.x];
}
__global__ __launch_bounds__(TPB) void paged_fork_kernel(const PagedPool p, int from, int to, int64_t len) {
    const int64_t i = (int64_t)blockIdx.x * TPB + threadIdx.x;
    const int h = blockIdx.y;
    if (h == 0 && i < (len + p.page - 1) >> p.shift) p.table[to * p.max_pages + i] = p.table[from * p.max_pages + i];
    if (p.weight && i < len) {
        const int64_t a = ((int64_t)from * p.heads + h) * p.max_len + i, b = ((int64_t)to * p.heads + h) * p.max_len + i;
        p.weight[b] = p.weight[a];
        p.pos[b] = p.pos[a];
    }
}

// ---- append --------------------------------------------------------------------------------------------------------
// A group of LPR lanes stores one key row and its value row.  int8 rows as kv_append_i8_kernel stores them: scale =
// max(max|x| / 127, 1e-8), codes round(x * (1 / scale)) away from zero at halves, within -127 .. 127; a wrong rounding
// is at most half a code.  VEC: 4 values per lane, else one value per lane and turn.
template <bool Q8, bool VEC, int LPR>
__device__ __forceinline__ void append_row(const float *__restrict__ src, void *cache, float *scales, int64_t row, int d, int l) {
    constexpr int N = VEC ? 1 : 4;  // pieces per lane (d <= 256)
    float4 x[N];
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (VEC) {
            if (4 * l < d) x[j] = *reinterpret_cast<const float4 *>(src + 4 * l);
        } else if (l + 64 * j < d) {
            x[j].x = src[l + 64 * j];
        }
        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w))));
    }
    if (!Q8) {
        float *dst = (float *)cache + row * d;
        if (VEC) {
            if (4 * l < d) *reinterpret_cast<float4 *>(dst + 4 * l) = x[0];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (l + 64 * j < d) dst[l + 64 * j] = x[j].x;
        }
        return;
    }
    mx = lanes_max<LPR>(mx);
    float scale = mx / 127.0f;
    if (!(scale > 1e-8f)) scale = 1e-8f;
    const float inv = 1.0f / scale;
    auto code = [&](float v) {
        float q = roundf(v * inv);
        q = q < -127.0f ? -127.0f : q > 127.0f ? 127.0f : q;
        return (int)q;
    };
    signed char *dst = (signed char *)cache + row * d;
    if (VEC) {
        if (4 * l < d)
            *reinterpret_cast<uint32_t *>(dst + 4 * l) = (uint32_t)(code(x[0].x) & 255) | (uint32_t)(code(x[0].y) & 255) << 8 |
                                                         (uint32_t)(code(x[0].z) & 255) << 16 | (uint32_t)(code(x[0].w) & 255) << 24;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (l + 64 * j < d) dst[l + 64 * j] = (signed char)code(x[j].x);
    }
    if (l == 0) scales[row] = scale;
}
template <bool Q8, bool VEC, int LPR>
__global__ __launch_bounds__(TPB) void paged_append_kernel(const PagedPool p, const PagedNew in, const PagedAppend a) {
    const uint32_t idx = blockIdx.x * (TPB / LPR) + threadIdx.x / LPR;
    const uint32_t ih = idx / (uint32_t)in.tokens, t = idx - ih * in.tokens;
    const uint32_t i = ih / (uint32_t)p.heads, h = ih - i * p.heads;
    if (i >= (uint32_t)a.n || t >= (uint32_t)a.count[i]) return;  // (whole groups leave)
    const int l = threadIdx.x % LPR;
    const int64_t at = (int64_t)a.len[i] + t;
    int32_t *entry = p.table + a.slot[i] * p.max_pages + (at >> p.shift);
    const int fresh = a.page[i];
    const int page = fresh >= 0 ? fresh : *entry;
    const int64_t row = row_of(p, page, h, (int)(at & (p.page - 1)));
    append_row<Q8, VEC, LPR>(in.k + i * in.k_seq + h * in.k_head + t * in.k_token, p.k, p.kscale, row, p.d, l);
    append_row<Q8, VEC, LPR>(in.v + i * in.v_seq + h * in.v_head + t * in.v_token, p.v, p.vscale, row, p.d, l);
    if (l == 0) {
        if (fresh >= 0 && h == 0) *entry = fresh;
        if (p.weight) {
            const int64_t track = ((int64_t)a.slot[i] * p.heads + h) * p.max_len + at;
            p.weight[track] = 0.f;
            p.pos[track] = a.seen[i] + (int)t;
        }
    }
}

// ---- attention of one new token ------------------------------------------------------------------------------------
// softmax(scale q k^T) v by the running maximum and sum, one pass over the rows.  A workgroup takes `chunk` positions
// of one sequence and key head, and with them up to G of the query heads that share it, so a row is read once for all
// of them.  Its four wavefronts walk the chunk in tiles; LPR lanes hold a row in 16-byte pieces (E values a lane), and
// every group of LPR lanes keeps a maximum, sum and output of its own, so nothing inside the loop crosses a group but
// the dot products.  The keys and the values of a tile (U rows each per group) are all requested before the first is
// used.  States meet at the end: inside the wavefront, then through LDS, then (more than one chunk) in
// paged_join_kernel, always in the same order.  Scores are kept in units of log2 e: the exponential is one v_exp_f32.
struct AttendArgs {
    PagedPool p;
    const float *q;
    float *out;
    float *part;    // [chunk of the launch][q_heads][d]: sums not yet divided (null: every sequence is one chunk)
    float2 *ml;     // [chunk of the launch][q_heads]: maximum and sum
    float *scores;  // accumulate: [sequence][q_heads][len], sequence i from element tokens_before[i] * q_heads on
    int n, q_heads, group, tiles_per_group, chunk;
    float scale;  // times log2 e
    int32_t slot[PAGED_BATCH], len[PAGED_BATCH];
    int32_t first[PAGED_BATCH + 1];          // first chunk of a sequence; INT_MAX behind the last sequence
    int32_t tokens_before[PAGED_BATCH];
};
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
            if (E * l < d) w = reinterpret_cast<const int4 *>((const char *)cache + row * d * (Q8 ? 1 : 4))[l];
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
template <bool VEC, int E>
__device__ __forceinline__ int column_of(int l, int e) { return VEC ? l * E + e : l + 64 * e; }

template <bool Q8, bool VEC, int LPR, int G, int U>
__global__ __launch_bounds__(TPB) void paged_attend_kernel(const AttendArgs a) {
    using Row = AttendRow<Q8, VEC>;
    constexpr int E = Row::E, RPP = 64 / LPR, TILE = RPP * U, WAVES = TPB / 64;
    extern __shared__ int32_t shared[];
    const PagedPool &p = a.p;
    const int d = p.d, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPR, sub = lane / LPR;
    const int b = blockIdx.x, i = sequence_of(a, b);
    const int h = blockIdx.y / a.tiles_per_group, g0 = (blockIdx.y % a.tiles_per_group) * G;
    const int t0 = (b - a.first[i]) * a.chunk, n = min(a.len[i] - t0, a.chunk);
    const int head0 = h * a.group + g0, heads = min(G, a.group - g0);
    // the chunk's pages
    const int p0 = t0 >> p.shift, pages = n > 0 ? ((t0 + n - 1) >> p.shift) - p0 + 1 : 0;
    for (int j = threadIdx.x; j < pages; j += TPB) shared[j] = p.table[a.slot[i] * p.max_pages + p0 + j];
    float qv[G][E], acc[G][E], m[G], sum[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        sum[g] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = column_of<VEC, E>(l, e);
            acc[g][e] = 0.f;
            qv[g][e] = g < heads && c < d ? a.q[((int64_t)i * a.q_heads + head0 + g) * d + c] : 0.f;
        }
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
        float s[G][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E];
            k[u].widen(x);
            const int t = base + u * RPP + sub;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float dot = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) dot += qv[g][e] * x[e];
                dot = lanes_sum<LPR>(dot) * a.scale;
                if (Q8) dot *= k[u].s;
                s[g][u] = t < n ? dot : -INFINITY;
                if (a.scores && t < n && l == 0 && g < heads)
                    a.scores[(int64_t)a.tokens_before[i] * a.q_heads + (int64_t)(head0 + g) * a.len[i] + t0 + t] = dot;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float top = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, s[g][u]);
            const float safe = top == -INFINITY ? 0.f : top;  // nothing yet, or nothing but scores of -inf
            const float fade = __builtin_amdgcn_exp2f(m[g] - safe);
            m[g] = top;
            sum[g] *= fade;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] *= fade;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[g][u] = __builtin_amdgcn_exp2f(s[g][u] - safe);
                sum[g] += s[g][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[E];
            v[u].widen(x);
            if (Q8) {
#pragma unroll
                for (int g = 0; g < G; ++g) s[g][u] *= v[u].s;
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[g][e] += s[g][u] * x[e];
        }
    }
    // the groups of a wavefront
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float mo = __shfl_xor(m[g], off, 64), so = __shfl_xor(sum[g], off, 64);
            const float top = fmaxf(m[g], mo), safe = top == -INFINITY ? 0.f : top;
            const float mine = __builtin_amdgcn_exp2f(m[g] - safe), theirs = __builtin_amdgcn_exp2f(mo - safe);
            m[g] = top;
            sum[g] = sum[g] * mine + so * theirs;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] = acc[g][e] * mine + __shfl_xor(acc[g][e], off, 64) * theirs;
        }
    }
    // the wavefronts of the workgroup: [G][WAVES][d], then [G][WAVES] maxima and sums
    __syncthreads();
    float *so = reinterpret_cast<float *>(shared), *sm = so + G * WAVES * d, *ss = sm + G * WAVES;
    if (sub == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = column_of<VEC, E>(l, e);
                if (c < d) so[(g * WAVES + wave) * d + c] = acc[g][e];
            }
            if (l == 0) { sm[g * WAVES + wave] = m[g]; ss[g * WAVES + wave] = sum[g]; }
        }
    }
    __syncthreads();
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
        if (!a.part) {
            a.out[((int64_t)i * a.q_heads + head0 + g) * d + c] = a.len[i] > 0 ? o / total : 0.f;
        } else {
            a.part[((int64_t)b * a.q_heads + head0 + g) * d + c] = o;
            if (c == 0) a.ml[(int64_t)b * a.q_heads + head0 + g] = make_float2(top, total);
        }
    }
}
// Joins the chunks: workgroups 0 .. n * q_heads - 1 an output row each; those behind add the probabilities of 1024
// positions of one key head to their weights (accumulate).
__global__ __launch_bounds__(TPB) void paged_join_kernel(const AttendArgs a, int blocks_per_head) {
    __shared__ float red[TPB / 64], out[TPB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = a.n * a.q_heads;
    if ((int)blockIdx.x < rows) {
        const int i = blockIdx.x / a.q_heads, head = blockIdx.x - i * a.q_heads, d = a.p.d;
        const int first = a.first[i], chunks = (a.len[i] + a.chunk - 1) / a.chunk;
        float top = -INFINITY;
        for (int c = threadIdx.x; c < chunks; c += TPB) top = fmaxf(top, a.ml[(int64_t)(first + c) * a.q_heads + head].x);
        top = lanes_max<64>(top);
        if (lane == 0) red[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float safe = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        for (int c = 0; c < chunks; ++c) {
            const float2 s = a.ml[(int64_t)(first + c) * a.q_heads + head];
            total += s.y * __builtin_amdgcn_exp2f(s.x - safe);
        }
        // columns over the threads, the chunks over TPB / columns groups of them
        const int cols = d < TPB ? d : TPB, groups = TPB / cols, col = threadIdx.x % cols, group = threadIdx.x / cols;
        float o = 0.f;
        if (group < groups)
            for (int c = group; c < chunks; c += groups) {
                const int64_t at = (int64_t)(first + c) * a.q_heads + head;
                o += a.part[at * d + col] * __builtin_amdgcn_exp2f(a.ml[at].x - safe);
            }
        out[threadIdx.x] = o;
        __syncthreads();
        if (threadIdx.x < (unsigned)cols) {
            for (int g = 1; g < groups; ++g) o += out[g * cols + col];
            a.out[(int64_t)blockIdx.x * d + col] = chunks > 0 ? o / total : 0.f;
        }
        return;
    }
    const int item = blockIdx.x - rows, ih = item / blocks_per_head, block = item - ih * blocks_per_head;
    const int i = ih / a.p.heads, h = ih - i * a.p.heads, len = a.len[i], t = block * 1024 + threadIdx.x;
    if (block * 1024 >= len) return;
    const int first = a.first[i], chunks = (len + a.chunk - 1) / a.chunk;
    const float *scores = a.scores + (int64_t)a.tokens_before[i] * a.q_heads;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < a.group; ++g) {
        const int head = h * a.group + g;
        float top = -INFINITY, total = 0.f;
        for (int c = lane; c < chunks; c += 64) {  // (every wavefront for itself)
            const float2 s = a.ml[(int64_t)(first + c) * a.q_heads + head];
            const float next = fmaxf(top, s.x), safe = next == -INFINITY ? 0.f : next;
            total = total * __builtin_amdgcn_exp2f(top - safe) + s.y * __builtin_amdgcn_exp2f(s.x - safe);
            top = next;
        }
        const float all = lanes_max<64>(top), safe = all == -INFINITY ? 0.f : all;
        total = lanes_sum<64>(total * __builtin_amdgcn_exp2f(top - safe));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (t + j * TPB < len) w[j] += __builtin_amdgcn_exp2f(scores[(int64_t)head * len + t + j * TPB] - safe) / total;
    }
    float *weight = a.p.weight + ((int64_t)a.slot[i] * a.p.heads + h) * a.p.max_len;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (t + j * TPB < len) weight[t + j * TPB] += w[j];
}

// ---- weights and positions -----------------------------------------------------------------------------------------
__global__ __launch_bounds__(TPB) void paged_add_weights_kernel(const PagedPool p, const PagedSeqs s, const float *__restrict__ w, int64_t width) {
    const int i = blockIdx.y / p.heads, h = blockIdx.y - i * p.heads;
    const int64_t t = (int64_t)blockIdx.x * TPB + threadIdx.x;
    if (t < s.len[i]) p.weight[((int64_t)s.slot[i] * p.heads + h) * p.max_len + t] += w[(int64_t)blockIdx.y * width + t];
}
__global__ __launch_bounds__(TPB) void paged_track_kernel(const PagedPool p, const PagedSeqs s, float *__restrict__ weights,
                                                          int32_t *__restrict__ positions, int64_t width) {
    const int i = blockIdx.y / p.heads, h = blockIdx.y - i * p.heads;
    const int64_t t = (int64_t)blockIdx.x * TPB + threadIdx.x;
    if (t >= width) return;
    const bool held = t < s.len[i];
    const int64_t from = ((int64_t)s.slot[i] * p.heads + h) * p.max_len + t;
    weights[(int64_t)blockIdx.y * width + t] = held ? p.weight[from] : 0.f;
    positions[(int64_t)blockIdx.y * width + t] = held ? p.pos[from] : -1;
}
// blockIdx.y: head, blockIdx.z: keys or values; a wavefront per row
__global__ __launch_bounds__(TPB) void paged_read_kernel(const PagedPool p, int slot, int64_t len, float *__restrict__ k, float *__restrict__ v) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= len) return;
    const int64_t row = row_of(p, p.table[slot * p.max_pages + (t >> p.shift)], blockIdx.y, (int)(t & (p.page - 1)));
    const void *cache = blockIdx.z ? p.v : p.k;
    float *dst = (blockIdx.z ? v : k) + ((int64_t)blockIdx.y * len + t) * p.d;
    for (int c = threadIdx.x & 63; c < p.d; c += 64)
        dst[c] = p.quantized ? (float)((const signed char *)cache)[row * p.d + c] * (blockIdx.z ? p.vscale : p.kscale)[row]
                             : ((const float *)cache)[row * p.d + c];
}

// ---- eviction ------------------------------------------------------------------------------------------------------
// One workgroup per (sequence, key head) finds the rows that stay.  They are the `budget` first by (recent tokens,
// weight, earlier position): a radix select on the weight as an ordered 32-bit key (recent rows above every key)
// finds the last key that stays, eight bits a pass; where only some of the rows with that key stay, a second select on
// the position tells which.  Then one pass in row order lists the freed places below the budget and the surviving rows
// behind it, and paged_move_kernel moves row j of the second list to place j of the first.  No row is both read and
// written, so the move needs no order and no second buffer, and it touches only what has to change place.
constexpr int SELECT_TPB = 1024;
struct EvictArgs {
    PagedPool p;
    int n, budget, recent, cap;
    int32_t *moves;  // [n][heads][2 * cap + 1]: count, places, sources
    int32_t slot[PAGED_BATCH], len[PAGED_BATCH], seen[PAGED_BATCH];
};
__device__ __forceinline__ uint32_t weight_key(float w, bool recent) {
    if (recent) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.0f);  // (-0 becomes +0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__global__ __launch_bounds__(SELECT_TPB) void paged_select_kernel(const EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[2];
    __shared__ int waves[2][SELECT_TPB / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = blockIdx.x / a.p.heads, h = blockIdx.x - i * a.p.heads, len = a.len[i];
    int32_t *out = a.moves + (int64_t)blockIdx.x * (2 * (int64_t)a.cap + 1);
    if (len <= a.budget) {
        if (tid == 0) out[0] = 0;
        return;
    }
    const int64_t at = ((int64_t)a.slot[i] * a.p.heads + h) * a.p.max_len;
    const float *w = a.p.weight + at;
    const int32_t *pos = a.p.pos + at;
    const int recent_from = a.seen[i] - a.recent;
    auto key_of = [&](int t) { return weight_key(w[t], pos[t] >= recent_from); };
    // Of the values value(t) with ok(t): the `want`-th in descending order (want >= 1), and how many of its equals
    // belong to the first `want`.
    auto select = [&](auto ok, auto value, uint32_t want, uint32_t &found, uint32_t &equals) {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int j = tid; j < 256; j += SELECT_TPB) hist[j] = 0;
            __syncthreads();
            for (int t = tid; t < len; t += SELECT_TPB)
                if (ok(t)) {
                    const uint32_t v = value(t);
                    if (shift == 24 || (v >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(v >> shift) & 255], 1u);
                }
            __syncthreads();
            if (wave == 0) {  // lane: bins 255 - 4 lane down to 252 - 4 lane, descending
                uint32_t c[4], mine = 0;
                for (int j = 0; j < 4; ++j) { c[j] = hist[255 - 4 * lane - j]; mine += c[j]; }
                uint32_t before = mine;
                for (int off = 1; off < 64; off <<= 1) {
                    const uint32_t x = __shfl_up(before, off, 64);
                    if (lane >= off) before += x;
                }
                before -= mine;
                for (int j = 0; j < 4; ++j) {
                    if (before < want && want <= before + c[j]) {
                        pick[0] = (uint32_t)(255 - 4 * lane - j);
                        pick[1] = want - before;
                    }
                    before += c[j];
                }
            }
            __syncthreads();
            prefix |= pick[0] << shift;
            want = pick[1];
            __syncthreads();
        }
        found = prefix;
        equals = want;
    };
    uint32_t key, ties;
    select([&](int) { return true; }, key_of, (uint32_t)a.budget, key, ties);
    // of the rows with that key the `ties` earliest stay: positions are below 2^31, so ~pos descends as they ascend
    uint32_t last, unused;
    select([&](int t) { return key_of(t) == key; }, [&](int t) { return ~(uint32_t)pos[t]; }, ties, last, unused);
    int holes = 0, movers = 0;
    for (int base = 0; base < len; base += SELECT_TPB) {
        const int t = base + tid;
        bool stays = false;
        if (t < len) {
            const uint32_t k = key_of(t);
            stays = k > key || (k == key && ~(uint32_t)pos[t] >= last);
        }
        const bool hole = t < a.budget && !stays, mover = t >= a.budget && t < len && stays;
        const unsigned long long hb = __ballot(hole), mb = __ballot(mover), below = (1ull << lane) - 1;
        if (lane == 0) { waves[0][wave] = __popcll(hb); waves[1][wave] = __popcll(mb); }
        __syncthreads();
        int ho = holes, mo = movers;
        for (int x = 0; x < SELECT_TPB / 64; ++x) {
            if (x < wave) { ho += waves[0][x]; mo += waves[1][x]; }
            holes += waves[0][x];
            movers += waves[1][x];
        }
        if (hole && ho + __popcll(hb & below) < a.cap) out[1 + ho + __popcll(hb & below)] = t;
        if (mover && mo + __popcll(mb & below) < a.cap) out[1 + a.cap + mo + __popcll(mb & below)] = t;
        __syncthreads();
    }
    if (tid == 0) out[0] = min(min(holes, movers), a.cap);
}
// A wavefront per move; blockIdx.y: (sequence, head).
__global__ __launch_bounds__(TPB) void paged_move_kernel(const EvictArgs a) {
    const PagedPool &p = a.p;
    const int i = blockIdx.y / p.heads, h = blockIdx.y - i * p.heads, lane = threadIdx.x & 63;
    const int32_t *moves = a.moves + (int64_t)blockIdx.y * (2 * (int64_t)a.cap + 1);
    const int j = blockIdx.x * (TPB / 64) + (threadIdx.x >> 6);
    if (j >= moves[0]) return;
    const int to = moves[1 + j], from = moves[1 + a.cap + j];
    const int32_t *table = p.table + a.slot[i] * p.max_pages;
    const int64_t dst = row_of(p, table[to >> p.shift], h, to & (p.page - 1)), src = row_of(p, table[from >> p.shift], h, from & (p.page - 1));
    const int bytes = p.d * (p.quantized ? 1 : 4);
    if (bytes % 16 == 0) {
        for (int c = lane; c < bytes / 16; c += 64) {
            const int4 k = reinterpret_cast<const int4 *>((const char *)p.k + src * bytes)[c], v = reinterpret_cast<const int4 *>((const char *)p.v + src * bytes)[c];
            reinterpret_cast<int4 *>((char *)p.k + dst * bytes)[c] = k;
            reinterpret_cast<int4 *>((char *)p.v + dst * bytes)[c] = v;
        }
    } else {
        for (int c = lane; c < bytes; c += 64) {
            ((char *)p.k)[dst * bytes + c] = ((const char *)p.k)[src * bytes + c];
            ((char *)p.v)[dst * bytes + c] = ((const char *)p.v)[src * bytes + c];
        }
    }
    if (lane == 0) {
        if (p.quantized) { p.kscale[dst] = p.kscale[src]; p.vscale[dst] = p.vscale[src]; }
        const int64_t at = ((int64_t)a.slot[i] * p.heads + h) * p.max_len;
        p.weight[at + to] = p.weight[at + from];
        p.pos[at + to] = p.pos[at + from];
    }
}

template <bool Q8, bool VEC, int LPR>
void launch_append(const PagedPool &p, const PagedNew &in, const PagedAppend &a) {
    const uint32_t rows = (uint32_t)a.n * p.heads * in.tokens;
    MNI_KERNEL_LAUNCH((paged_append_kernel<Q8, VEC, LPR>), dim3((rows + TPB / LPR - 1) / (TPB / LPR)), dim3(TPB), 0, ctx().stream, p, in, a);
}
template <bool Q8, bool VEC, int LPR, int G, int U>
void launch_attend(const AttendArgs &a, int chunks) {
    const int pages = a.chunk / a.p.page + 2;
    const int merge = G * (TPB / 64) * (a.p.d + 2);
    const size_t lds = (size_t)(pages > merge ? pages : merge) * 4;
    MNI_KERNEL_LAUNCH((paged_attend_kernel<Q8, VEC, LPR, G, U>), dim3((unsigned)chunks, (unsigned)(a.p.heads * a.tiles_per_group)), dim3(TPB), lds,
                      ctx().stream, a);
}
template <bool Q8, bool VEC, int LPR>
void launch_attend_heads(AttendArgs &a, int chunks, int g) {
    a.tiles_per_group = (a.group + g - 1) / g;
    if (g == 1) launch_attend<Q8, VEC, LPR, 1, Q8 ? 4 : 8>(a, chunks);
    else if (g == 2) launch_attend<Q8, VEC, LPR, 2, 4>(a, chunks);
    else launch_attend<Q8, VEC, LPR, 4, 4>(a, chunks);
}

}  // namespace

int k_paged_table(const PagedPool &p, const PagedTableWrite &w) {
    if (w.n <= 0) return MNI_OK;
    MNI_KERNEL_LAUNCH(paged_table_kernel, dim3(1), dim3(TPB), 0, ctx().stream, p.table, w);
    return check_launch("paged_table");
}
int k_paged_copy(const PagedPool &p, const PagedCopies &c) {
    if (c.n <= 0) return MNI_OK;
    MNI_KERNEL_LAUNCH(paged_copy_kernel, dim3((unsigned)c.n, p.quantized ? 4 : 2), dim3(TPB), 0, ctx().stream, p, c);
    return check_launch("paged_copy");
}
int k_paged_fork(const PagedPool &p, int32_t from, int32_t to, int64_t len) {
    if (len <= 0) return MNI_OK;
    const int heads = p.weight ? p.heads : 1;
    MNI_KERNEL_LAUNCH(paged_fork_kernel, dim3((unsigned)((len + TPB - 1) / TPB), (unsigned)heads), dim3(TPB), 0, ctx().stream, p, from, to, len);
    return check_launch("paged_fork");
}
int k_paged_append(const PagedPool &p, const PagedNew &in, const PagedAppend &a) {
    if (a.n <= 0 || in.tokens <= 0) return MNI_OK;
    const bool vec = p.d % 4 == 0 && (((uintptr_t)in.k | (uintptr_t)in.v) & 15) == 0 &&
                     ((in.k_seq | in.k_head | in.k_token | in.v_seq | in.v_head | in.v_token) & 3) == 0;
    if (!vec) {
        if (p.quantized) launch_append<true, false, 64>(p, in, a);
        else launch_append<false, false, 64>(p, in, a);
    } else if (p.quantized) {
        if (p.d <= 64) launch_append<true, true, 16>(p, in, a);
        else if (p.d <= 128) launch_append<true, true, 32>(p, in, a);
        else launch_append<true, true, 64>(p, in, a);
    } else {
        if (p.d <= 64) launch_append<false, true, 16>(p, in, a);
        else if (p.d <= 128) launch_append<false, true, 32>(p, in, a);
        else launch_append<false, true, 64>(p, in, a);
    }
    return check_launch("paged_append");
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
    a.n = s.n;
    a.q_heads = q_heads;
    a.group = q_heads / p.heads;
    a.scale = scale * LOG2E;
    const bool vec = p.d % (p.quantized ? 16 : 4) == 0 && ((uintptr_t)q & 15) == 0;
    const int g = a.group == 1 ? 1 : a.group == 2 ? 2 : 4;
    // about four workgroups per CU, chunks in whole turns of the four wavefronts
    int64_t tokens = 0, longest = 0;
    for (int i = 0; i < s.n; ++i) {
        tokens += s.len[i];
        if (s.len[i] > longest) longest = s.len[i];
    }
    const int64_t per_token = (int64_t)p.heads * ((a.group + g - 1) / g);
    int64_t chunk = tokens * per_token / (4 * 256);
    chunk = (chunk + 127) / 128 * 128;
    if (chunk < 128) chunk = 128;
    if (chunk > 4096) chunk = 4096;
    a.chunk = (int)chunk;
    int chunks = 0;
    int64_t before = 0;
    bool several = false;
    for (int i = 0; i < PAGED_BATCH; ++i) {
        a.slot[i] = i < s.n ? s.slot[i] : 0;
        a.len[i] = i < s.n ? s.len[i] : 0;
        a.first[i] = i < s.n ? chunks : INT_MAX;
        a.tokens_before[i] = (int32_t)before;
        if (i < s.n) {
            const int c = s.len[i] > 0 ? (int)((s.len[i] + chunk - 1) / chunk) : 1;  // an empty sequence: one that writes zeros
            several = several || c > 1;
            chunks += c;
            before += s.len[i];
            if (before > INT_MAX) return set_error(MNI_ERR_INVALID, "paged cache attend: more than 2^31 positions in one call");
        }
    }
    a.first[s.n] = s.n < PAGED_BATCH ? INT_MAX : INT_MAX;
    for (int i = s.n; i <= PAGED_BATCH; ++i) a.first[i] = INT_MAX;
    void *part = nullptr, *ml = nullptr, *scores = nullptr;
    int rc = MNI_OK;
    if (several || accumulate) {
        rc = dev_alloc(&part, (size_t)chunks * q_heads * p.d * sizeof(float));
        if (rc == MNI_OK) rc = dev_alloc(&ml, (size_t)chunks * q_heads * sizeof(float2));
        if (rc == MNI_OK && accumulate) rc = dev_alloc(&scores, (size_t)(before > 0 ? before : 1) * q_heads * sizeof(float));
        a.part = (float *)part;
        a.ml = (float2 *)ml;
        a.scores = (float *)scores;
    }
    if (rc == MNI_OK) {
        const int pieces = vec ? p.d / (p.quantized ? 16 : 4) + (p.d % (p.quantized ? 16 : 4) != 0) : 64;
        if (!vec) {
            if (p.quantized) launch_attend_heads<true, false, 64>(a, chunks, g);
            else launch_attend_heads<false, false, 64>(a, chunks, g);
        } else if (p.quantized) {
            if (pieces <= 4) launch_attend_heads<true, true, 4>(a, chunks, g);
            else if (pieces <= 8) launch_attend_heads<true, true, 8>(a, chunks, g);
            else launch_attend_heads<true, true, 16>(a, chunks, g);
        } else {
            if (pieces <= 8) launch_attend_heads<false, true, 8>(a, chunks, g);
            else if (pieces <= 16) launch_attend_heads<false, true, 16>(a, chunks, g);
            else if (pieces <= 32) launch_attend_heads<false, true, 32>(a, chunks, g);
            else launch_attend_heads<false, true, 64>(a, chunks, g);
        }
        rc = check_launch("paged_attend");
    }
    if (rc == MNI_OK && a.part) {
        const int per_head = accumulate ? (int)((longest + 1023) / 1024) : 0;
        const int64_t blocks = (int64_t)s.n * q_heads + (int64_t)s.n * p.heads * per_head;
        MNI_KERNEL_LAUNCH(paged_join_kernel, dim3((unsigned)blocks), dim3(TPB), 0, ctx().stream, a, per_head);
        rc = check_launch("paged_join");
    }
    if (part) dev_free(part);
    if (ml) dev_free(ml);
    if (scores) dev_free(scores);
    return rc;
}

int k_paged_add_weights(const PagedPool &p, const PagedSeqs &s, const float *w, int64_t width) {
    int64_t longest = 0;
    for (int i = 0; i < s.n; ++i)
        if (s.len[i] > longest) longest = s.len[i];
    if (longest == 0) return MNI_OK;
    MNI_KERNEL_LAUNCH(paged_add_weights_kernel, dim3((unsigned)((longest + TPB - 1) / TPB), (unsigned)(s.n * p.heads)), dim3(TPB), 0, ctx().stream, p, s, w,
                      width);
    return check_launch("paged_add_weights");
}
int k_paged_track(const PagedPool &p, const PagedSeqs &s, float *weights, int32_t *positions, int64_t width) {
    if (s.n <= 0 || width <= 0) return MNI_OK;
    MNI_KERNEL_LAUNCH(paged_track_kernel, dim3((unsigned)((width + TPB - 1) / TPB), (unsigned)(s.n * p.heads)), dim3(TPB), 0, ctx().stream, p, s, weights,
                      positions, width);
    return check_launch("paged_track");
}
int k_paged_read(const PagedPool &p, int32_t slot, int64_t len, float *k, float *v) {
    if (len <= 0) return MNI_OK;
    MNI_KERNEL_LAUNCH(paged_read_kernel, dim3((unsigned)((len + 3) / 4), (unsigned)p.heads, 2), dim3(TPB), 0, ctx().stream, p, (int)slot, len, k, v);
    return check_launch("paged_read");
}
int k_paged_evict(const PagedPool &p, const PagedSeqs &s, const int32_t *seen, int budget, int recent) {
    EvictArgs a;
    a.p = p;
    a.n = s.n;
    a.budget = budget;
    a.recent = recent;
    int64_t longest = 0;
    for (int i = 0; i < PAGED_BATCH; ++i) {
        a.slot[i] = i < s.n ? s.slot[i] : 0;
        a.len[i] = i < s.n ? s.len[i] : 0;
        a.seen[i] = i < s.n ? seen[i] : 0;
        if (a.len[i] > longest) longest = a.len[i];
    }
    const int64_t behind = longest - budget;
    if (s.n <= 0 || behind <= 0 || budget <= 0) return MNI_OK;
    a.cap = (int)(behind < budget ? behind : budget);  // at most so many rows change place
    void *moves = nullptr;
    MNI_TRY(dev_alloc(&moves, (size_t)s.n * p.heads * (2 * (size_t)a.cap + 1) * sizeof(int32_t)));
    a.moves = (int32_t *)moves;
    MNI_KERNEL_LAUNCH(paged_select_kernel, dim3((unsigned)(s.n * p.heads)), dim3(SELECT_TPB), 0, ctx().stream, a);
    int rc = check_launch("paged_select");
    if (rc == MNI_OK) {
        MNI_KERNEL_LAUNCH(paged_move_kernel, dim3((unsigned)((a.cap + 3) / 4), (unsigned)(s.n * p.heads)), dim3(TPB), 0, ctx().stream, a);
        rc = check_launch("paged_move");
    }
    dev_free(moves);
    return rc;
}

}  // namespace mni
