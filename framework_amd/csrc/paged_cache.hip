// Kernels of the paged key-value cache (mni_paged_cache_*): append, copies, eviction by accumulated weight (attention over
// its pages is in paged_attend.hip).  All of them are bound by memory.
#include "lanes.h"
#include "paged_cache.h"

namespace mni {
namespace {

constexpr int TPB = 256;
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---- page copies, forks -----------------------------------------------------------------------------
// blockIdx.x: the copy, blockIdx.y: keys, values, key scales, value scales.  A page is one contiguous block, copied in
// pieces of 16 KB (1 MB of keys and 1 of values: 3.6 us, launch-bound).
__global__ __launch_bounds__(TPB) void paged_copy_kernel(const PagedPool p, const PagedCopies c) {
    const int what = blockIdx.y;
    const int64_t rows = (int64_t)p.heads * p.page, unit = what >= 2 || !p.quantized ? 4 : 1;
    const int64_t bytes = rows * (what >= 2 ? 1 : p.d) * unit;
    char *base = (char *)(what == 0 ? p.k : what == 1 ? p.v : what == 2 ? (void *)p.kscale : (void *)p.vscale);
    const char *src = base + c.from[blockIdx.x] * bytes;
    char *dst = base + c.to[blockIdx.x] * bytes;
    const int64_t first = (int64_t)blockIdx.z * TPB + threadIdx.x, step = (int64_t)gridDim.z * TPB;
    if (bytes % 16 == 0) {
        for (int64_t i = first; i < bytes / 16; i += step) reinterpret_cast<int4 *>(dst)[i] = reinterpret_cast<const int4 *>(src)[i];
    } else {
        for (int64_t i = first; i < bytes; i += step) dst[i] = src[i];
    }
    if (what == 0 && first == 0) p.table[c.at[blockIdx.x]] = c.to[blockIdx.x];
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
// A group of LPR lanes stores one key row and its value row.  int8: scale = max(max|x| * (1 / 127), 1e-8), codes
// round(x * (1 / scale)), halves away from zero: a stored value is at most half a scale off, and no code leaves -127 .. 127
// (the largest is 127 to three roundings).  A row that holds an infinity or a NaN gets that for its scale and codes of 0, so
// that all of it reads as NaN, in attention too; the maximum is taken of the bits, where a float maximum would lose the NaN.
// (The contiguous cache divides by 127; the two scales differ by one rounding.)
// VEC: 4 values per lane, else one value per lane and turn.  Bound by bandwidth: 134 MB of fp32 rows read and written in 46
// us (5.8 TB/s, the rate of a large copy), 31 MB stored as 8 MB of int8 rows in 9.5.
template <bool VEC>
struct AppendRow {
    static constexpr int N = VEC ? 1 : 4;  // pieces per lane (d <= 256)
    float4 x[N];
    __device__ __forceinline__ void load(const float *__restrict__ src, int d, int l) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (VEC) {  // (the lanes behind the row repeat its last piece: no branch before the loads)
                x[j] = *reinterpret_cast<const float4 *>(src + min(4 * l, d - 4));
            } else if (l + 64 * j < d) {
                x[j].x = src[l + 64 * j];
            }
        }
    }
    template <bool Q8, int LPR>
    __device__ __forceinline__ void store(void *cache, float *scales, int64_t row, int d, int l) const {
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
        auto bits = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };  // of |v|
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) top = max(top, max(max(bits(x[j].x), bits(x[j].y)), max(bits(x[j].z), bits(x[j].w))));
        top = lanes_max_bits<LPR>(top);
        const bool finite = top < 0x7f800000u;
        float scale = __uint_as_float(top) * (1.0f / 127.0f);
        if (scale < 1e-8f) scale = 1e-8f;  // (a NaN stays)
        const float inv = 1.0f / scale;
        // halves away from zero: the whole part of y and, towards its sign, the largest value below a half (what round() gives
        // for every |y| up to 128; the product is rounded before the sum, which a fused multiply-add would not do)
        auto code = [&](float v) {
#pragma clang fp contract(off)
            const float y = v * inv;
            return (int)(y + copysignf(0.49999997f, y));
        };
        signed char *dst = (signed char *)cache + row * d;
        if (VEC) {
            if (4 * l < d)
                *reinterpret_cast<uint32_t *>(dst + 4 * l) =
                    finite ? __builtin_amdgcn_perm((uint32_t)code(x[0].w), (uint32_t)code(x[0].z), 0x04000c0c) |
                                 __builtin_amdgcn_perm((uint32_t)code(x[0].y), (uint32_t)code(x[0].x), 0x0c0c0400)
                           : 0u;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (l + 64 * j < d) dst[l + 64 * j] = (signed char)(finite ? code(x[j].x) : 0);
        }
        if (l == 0) scales[row] = scale;
    }
};
// The page of position `at` of sequence i, and whether it is a new one.
__device__ __forceinline__ int page_of(const PagedPool &p, const PagedAppend &a, int i, int64_t at, bool &fresh) {
    fresh = a.page[i] >= 0;
    return fresh ? a.page[i] : p.table[a.slot[i] * p.max_pages + (at >> p.shift)];
}
__device__ __forceinline__ int page_of(const PagedPool &p, const PagedPrompt &a, int i, int64_t at, bool &fresh) {
    const int index = (int)(at >> p.shift);
    fresh = index >= a.had[i];
    return fresh ? a.pages[a.first[i] + index - a.had[i]] : p.table[a.slot[i] * p.max_pages + index];
}
// A row of keys and values per group of LPR lanes.  (Four rows a group, all asked for before the first is stored: 68
// against 46 us on 134 MB of fp32 rows, 13 against 10 on 29 MB of them stored as int8.)
template <bool Q8, bool VEC, int LPR, class Batch>
__global__ __launch_bounds__(TPB) void paged_append_kernel(const PagedPool p, const PagedNew in, const Batch a, uint32_t first) {
    const uint32_t idx = (first + blockIdx.x) * (TPB / LPR) + threadIdx.x / LPR;  // (at most 2^31 rows and a workgroup's)
    const uint32_t ih = idx / (uint32_t)in.tokens, t = idx - ih * in.tokens;
    const uint32_t i = ih / (uint32_t)p.heads, h = ih - i * p.heads;
    if (i >= (uint32_t)a.n || t >= (uint32_t)a.count[i]) return;  // (whole groups leave)
    const int l = threadIdx.x % LPR;
    AppendRow<VEC> k, v;
    k.load(in.k + i * in.k_seq + h * in.k_head + t * in.k_token, p.d, l);
    v.load(in.v + i * in.v_seq + h * in.v_head + t * in.v_token, p.d, l);
    const int64_t at = (int64_t)a.len[i] + t;
    bool fresh;
    const int page = page_of(p, a, (int)i, at, fresh), off = (int)(at & (p.page - 1));
    const int64_t row = row_of(p, page, h, off);
    k.template store<Q8, LPR>(p.k, p.kscale, row, p.d, l);
    v.template store<Q8, LPR>(p.v, p.vscale, row, p.d, l);
    if (l != 0) return;
    if (fresh && h == 0 && off == 0) p.table[a.slot[i] * p.max_pages + (at >> p.shift)] = page;
    if (p.weight) {
        const int64_t track = ((int64_t)a.slot[i] * p.heads + h) * p.max_len + at;
        p.weight[track] = 0.f;
        p.pos[track] = a.seen[i] + t;
    }
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
    const void *cache = blockIdx.z ? p.v : p.k;
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < len; t += (int64_t)gridDim.x * 4) {
        const int64_t row = row_of(p, p.table[slot * p.max_pages + (t >> p.shift)], blockIdx.y, (int)(t & (p.page - 1)));
        float *dst = (blockIdx.z ? v : k) + ((int64_t)blockIdx.y * len + t) * p.d;
        for (int c = threadIdx.x & 63; c < p.d; c += 64)
            dst[c] = p.quantized ? (float)((const signed char *)cache)[row * p.d + c] * (blockIdx.z ? p.vscale : p.kscale)[row]
                                 : ((const float *)cache)[row * p.d + c];
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------------
// One workgroup per (sequence, key head) finds the rows that stay: the `budget` first by (recent tokens, weight, earlier
// position).  The weight becomes an ordered 32-bit key (recent rows above every key), and the last key that stays is found
// by its digits of eight bits from the highest on, each from a histogram of the keys that share the digits before; where
// only some of the rows with that key stay, the same search on the position tells which.  A thread holds its keys in
// registers (up to 16384 rows: 27 us there, 36 read again for every digit; with 32 keys a thread the registers spill, 56
// against 52 us at 24000 rows), every digit has a histogram of its
// own, cleared at the start, and every wavefront reads it for itself: one barrier a digit.  (Two bits a turn by ballots, with
// nothing to collide on, took 35 us on 256 x 4608 rows.)  Then one pass in row order lists the freed places below the
// budget and the surviving rows behind it, and row j of the second list moves to place j of the first.
// No row is both read and written, so the move needs no order and no second buffer, and it touches only what has to
// change place.  Where little moves (32 KB of keys a workgroup at most) the workgroup does it itself, with the lists in LDS;
// more is moved by a launch of its own, with the whole chip's loads in flight (from the start of the first to the end of the
// last, us: 48 workgroups x 77 rows of 256 bytes 10.4, in two launches 15.5; 256 x 64 of 512 bytes 16.8 and 17.2; 8 x 128 of
// 512 16.4 and 15.8; 32 x 1024 of 64 24.1 and 21.1).
constexpr int SELECT_TPB = 1024;
constexpr int SELECT_LIST = 1024;  // moves whose lists take the place of the histograms
struct EvictArgs {
    PagedPool p;
    int n, budget, recent, cap, lanes_log2;
    int32_t *moves;  // [n][heads][2 * cap + 1]: count, places, sources; null: the selection moves the rows itself
    int32_t slot[PAGED_BATCH], len[PAGED_BATCH], seen[PAGED_BATCH];
};
__device__ __forceinline__ uint32_t weight_key(float w, bool recent) {
    const uint32_t u = __float_as_uint(w + 0.0f);  // (-0 becomes +0)
    const uint32_t key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return recent ? 0xffffffffu : w != w ? 0xfffffffeu : key;
}
// Row `from` of a head takes the place `to`, by `lanes` lanes.
__device__ __forceinline__ void move_row(const EvictArgs &a, int i, int h, int to, int from, int lane, int lanes) {
    const PagedPool &p = a.p;
    const int32_t *table = p.table + a.slot[i] * p.max_pages;
    const int64_t dst = row_of(p, table[to >> p.shift], h, to & (p.page - 1)), src = row_of(p, table[from >> p.shift], h, from & (p.page - 1));
    const int bytes = p.d * (p.quantized ? 1 : 4);
    if (bytes % 16 == 0) {
        for (int c = lane; c < bytes / 16; c += lanes) {
            const i32x4 k = reinterpret_cast<const i32x4 *>((const char *)p.k + src * bytes)[c], v = reinterpret_cast<const i32x4 *>((const char *)p.v + src * bytes)[c];
            __builtin_nontemporal_store(k, reinterpret_cast<i32x4 *>((char *)p.k + dst * bytes) + c);
            __builtin_nontemporal_store(v, reinterpret_cast<i32x4 *>((char *)p.v + dst * bytes) + c);
        }
    } else {
        for (int c = lane; c < bytes; c += lanes) {
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
template <int KEYS>  // rows a thread holds: up to KEYS * SELECT_TPB in all; 0: none, they are read every time
__global__ __launch_bounds__(SELECT_TPB) void paged_select_kernel(const EvictArgs a) {
    constexpr int WAVES = SELECT_TPB / 64;
    __shared__ uint32_t hist[8][256];
    __shared__ int waves[2][WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = blockIdx.x / a.p.heads, h = blockIdx.x - i * a.p.heads, len = a.len[i];
    int32_t *out = a.moves ? a.moves + (int64_t)blockIdx.x * (2 * (int64_t)a.cap + 1) : nullptr;
    if (len <= a.budget) {
        if (tid == 0 && out) out[0] = 0;
        return;
    }
    const int64_t at = ((int64_t)a.slot[i] * a.p.heads + h) * a.p.max_len;
    const float *w = a.p.weight + at;
    const int32_t *pos = a.p.pos + at;
    const int recent_from = a.seen[i] - a.recent, top = a.seen[i];  // positions are below `top`
    for (int j = tid; j < 8 * 256; j += SELECT_TPB) hist[j >> 8][j & 255] = 0;
    uint32_t held[KEYS ? KEYS : 1];
    if (KEYS) {  // (all asked for before the first is looked at)
        float hw[KEYS ? KEYS : 1];
        int hp[KEYS ? KEYS : 1];
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
            if (j * SELECT_TPB < len) {
                const int t = min(tid + j * SELECT_TPB, len - 1);
                hw[j] = w[t];
                hp[j] = pos[t];
            }
#pragma unroll
        for (int j = 0; j < KEYS; ++j) held[j] = j * SELECT_TPB < len ? weight_key(hw[j], hp[j] >= recent_from) : 0;
    }
    __syncthreads();
    // f(key, row) for every row this thread looks at; whole wavefronts call it together
    auto each = [&](auto f) {
        if (KEYS) {
#pragma unroll
            for (int j = 0; j < KEYS; ++j)
                if (j * SELECT_TPB < len) f(held[j], tid + j * SELECT_TPB);
        } else {
            for (int base = 0; base < len; base += SELECT_TPB) {
                const int t = base + tid;
                f(weight_key(w[min(t, len - 1)], pos[min(t, len - 1)] >= recent_from), t);
            }
        }
    };
    // Of the values value(key, row) of the rows with takes(key, row): the `want`-th in descending order.  `equals`: how many
    // rows with that value are among the first `want`, `all`: how many there are.
    int slot = 0;
    auto search = [&](int digits, uint32_t want, auto takes, auto value, uint32_t &equals, uint32_t &all) {
        uint32_t found = 0;
#pragma unroll 1
        for (int shift = 8 * (digits - 1); shift >= 0; shift -= 8, ++slot) {
            each([&](uint32_t key, int t) {
                const uint32_t v = value(key, t);
                if (t < len && takes(key, t) && ((v ^ found) >> shift) < 256) atomicAdd(&hist[slot][(v >> shift) & 255], 1u);
            });
            __syncthreads();
            // lane: digits 255 - 4 lane down to 252 - 4 lane
            const uint4 h4 = *reinterpret_cast<const uint4 *>(&hist[slot][252 - 4 * lane]);
            const uint32_t c[4] = {h4.w, h4.z, h4.y, h4.x};
            uint32_t before = c[0] + c[1] + c[2] + c[3];
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t x = __shfl_up(before, off, 64);
                if (lane >= off) before += x;
            }
            const int at_lane = __ffsll((unsigned long long)__ballot(before >= want)) - 1;
            before -= c[0] + c[1] + c[2] + c[3];
            uint32_t digit = 0, rest = 0, count = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < want && want <= before + c[j]) {
                    digit = (uint32_t)(255 - 4 * lane - j);
                    rest = want - before;
                    count = c[j];
                }
                before += c[j];
            }
            found |= (uint32_t)__builtin_amdgcn_readlane((int)digit, at_lane) << shift;
            want = (uint32_t)__builtin_amdgcn_readlane((int)rest, at_lane);
            all = (uint32_t)__builtin_amdgcn_readlane((int)count, at_lane);
        }
        equals = want;
        return found;
    };
    uint32_t ties, equal, late = 0, unused;
    const uint32_t key = search(4, (uint32_t)a.budget, [](uint32_t, int) { return true; }, [](uint32_t k, int) { return k; }, ties, equal);
    if (ties < equal) {  // of the rows with that key the earliest stay: those of a value top - 1 - position of at least `late`
        const int digits = (39 - __clz(top > 1 ? top - 1 : 1)) / 8;
        late = search(digits, ties, [&](uint32_t k, int) { return k == key; }, [&](uint32_t, int t) { return (uint32_t)(top - 1 - pos[min(t, len - 1)]); }, unused,
                      unused);
    }
    __syncthreads();  // (the histograms are read no more: they become the lists)
    int32_t *places = out ? out + 1 : reinterpret_cast<int32_t *>(&hist[0][0]), *sources = places + a.cap;
    int holes = 0, movers = 0;
    each([&](uint32_t k, int t) {
        const bool stays = t < len && (k > key || (k == key && (late == 0 || (uint32_t)(top - 1 - pos[min(t, len - 1)]) >= late)));
        const bool hole = t < a.budget && !stays, mover = t >= a.budget && stays;
        const unsigned long long hb = __ballot(hole), mb = __ballot(mover), below = (1ull << lane) - 1;
        if (lane == 0) { waves[0][wave] = __popcll(hb); waves[1][wave] = __popcll(mb); }
        __syncthreads();
        int ho = holes, mo = movers;
        for (int x = 0; x < WAVES; ++x) {
            if (x < wave) { ho += waves[0][x]; mo += waves[1][x]; }
            holes += waves[0][x];
            movers += waves[1][x];
        }
        if (hole && ho + __popcll(hb & below) < a.cap) places[ho + __popcll(hb & below)] = t;
        if (mover && mo + __popcll(mb & below) < a.cap) sources[mo + __popcll(mb & below)] = t;
        __syncthreads();
    });
    const int count = min(min(holes, movers), a.cap);
    if (out) {
        if (tid == 0) out[0] = count;
        return;
    }
    const int lanes = 1 << a.lanes_log2;
#pragma unroll 2
    for (int j = tid >> a.lanes_log2; j < count; j += SELECT_TPB >> a.lanes_log2) move_row(a, i, h, places[j], sources[j], tid & (lanes - 1), lanes);
}
// As many lanes per move as a row has 16-byte pieces, rounded up to a power of two (other rows: 64); blockIdx.y: (sequence,
// head).  32 x 4096 moves of 64-byte rows take 7 us so, 26 at a wavefront each; 256 x 512 of 512 bytes 32 and 37.  Rows are
// stored past the caches (nontemporal): left in the last-level cache they are written back under the next attention's
// reads (1.07 GB of rows behind 230 MB of moves and appends: 214 us instead of 162).
__global__ __launch_bounds__(TPB) void paged_move_kernel(const EvictArgs a) {
    const int i = blockIdx.y / a.p.heads, h = blockIdx.y - i * a.p.heads, lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int32_t *moves = a.moves + (int64_t)blockIdx.y * (2 * (int64_t)a.cap + 1);
    const int rows = TPB >> a.lanes_log2, count = moves[0];
    for (int j = blockIdx.x * rows + (threadIdx.x >> a.lanes_log2); j < count; j += gridDim.x * rows)  // (once, but in the largest grid)
        move_row(a, i, h, moves[1 + j], moves[1 + a.cap + j], lane, lanes);
}

int launch_allowed(const char *what) {  // (see mni_rocm_test_fail_paged_launch)
    int64_t &left = ctx().paged_launch_fails_in;
    if (left > 0 && --left == 0) return set_error(MNI_ERR_HIP, "launch of %s failed: a test asked for it", what);
    return MNI_OK;
}
template <bool Q8, bool VEC, int LPR, class Batch>
void launch_append(const PagedPool &p, const PagedNew &in, const Batch &a) {
    const int64_t rows = (int64_t)a.n * p.heads * in.tokens, blocks = (rows + TPB / LPR - 1) / (TPB / LPR);
    for (int64_t first = 0; first < blocks; first += most_blocks(TPB)) {
        const int64_t some = blocks - first < most_blocks(TPB) ? blocks - first : most_blocks(TPB);
        MNI_KERNEL_LAUNCH((paged_append_kernel<Q8, VEC, LPR, Batch>), dim3((unsigned)some), dim3(TPB), 0, ctx().stream, p, in, a, (uint32_t)first);
    }
}
template <class Batch>
int paged_append(const PagedPool &p, const PagedNew &in, const Batch &a) {
    if (a.n <= 0 || in.tokens <= 0) return MNI_OK;
    MNI_TRY(launch_allowed("paged_append"));
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

}  // namespace

int k_paged_copy(const PagedPool &p, const PagedCopies &c) {
    if (c.n <= 0) return MNI_OK;
    MNI_TRY(launch_allowed("paged_copy"));
    const int64_t bytes = (int64_t)p.heads * p.page * p.d * (p.quantized ? 1 : 4), parts = (bytes + 16383) / 16384;
    MNI_KERNEL_LAUNCH(paged_copy_kernel, dim3((unsigned)c.n, p.quantized ? 4 : 2, (unsigned)(parts < 1024 ? parts : 1024)), dim3(TPB), 0, ctx().stream, p, c);
    return check_launch("paged_copy");
}
int k_paged_fork(const PagedPool &p, int32_t from, int32_t to, int64_t len) {
    if (len <= 0) return MNI_OK;
    const int heads = p.weight ? p.heads : 1;
    MNI_KERNEL_LAUNCH(paged_fork_kernel, dim3((unsigned)((len + TPB - 1) / TPB), (unsigned)heads), dim3(TPB), 0, ctx().stream, p, from, to, len);
    return check_launch("paged_fork");
}
int k_paged_append(const PagedPool &p, const PagedNew &in, const PagedAppend &a) { return paged_append(p, in, a); }
int k_paged_append(const PagedPool &p, const PagedNew &in, const PagedPrompt &a) { return paged_append(p, in, a); }

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
    const int64_t blocks = (len + 3) / 4;
    MNI_KERNEL_LAUNCH(paged_read_kernel, dim3((unsigned)(blocks < most_blocks(TPB) ? blocks : most_blocks(TPB)), (unsigned)p.heads, 2), dim3(TPB), 0, ctx().stream, p, (int)slot, len, k, v);
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
    MNI_TRY(launch_allowed("paged_select"));
    a.cap = (int)(behind < budget ? behind : budget);  // at most so many rows change place
    const int bytes = p.d * (p.quantized ? 1 : 4);
    a.lanes_log2 = 0;
    while (a.lanes_log2 < 6 && (bytes % 16 || (16 << a.lanes_log2) < bytes)) ++a.lanes_log2;
    const bool fused = a.cap <= SELECT_LIST && (int64_t)a.cap * bytes <= 32768;
    void *moves = nullptr;
    if (!fused) MNI_TRY(dev_alloc(&moves, (size_t)s.n * p.heads * (2 * (size_t)a.cap + 1) * sizeof(int32_t)));
    a.moves = (int32_t *)moves;
    const dim3 grid((unsigned)(s.n * p.heads));
    if (longest <= 8 * SELECT_TPB) MNI_KERNEL_LAUNCH(paged_select_kernel<8>, grid, dim3(SELECT_TPB), 0, ctx().stream, a);
    else if (longest <= 16 * SELECT_TPB) MNI_KERNEL_LAUNCH(paged_select_kernel<16>, grid, dim3(SELECT_TPB), 0, ctx().stream, a);
    else MNI_KERNEL_LAUNCH(paged_select_kernel<0>, grid, dim3(SELECT_TPB), 0, ctx().stream, a);
    int rc = check_launch("paged_select");
    if (rc == MNI_OK && !fused) {
        const int per_block = TPB >> a.lanes_log2;
        const int64_t blocks = (a.cap + per_block - 1) / per_block;
        MNI_KERNEL_LAUNCH(paged_move_kernel, dim3((unsigned)(blocks < most_blocks(TPB) ? blocks : most_blocks(TPB)), (unsigned)(s.n * p.heads)), dim3(TPB), 0,
                          ctx().stream, a);
        rc = check_launch("paged_move");
    }
    if (moves) dev_free(moves);
    return rc;
}

}  // namespace mni
