// Norm of queries and keys for each head with the rotation of their positions in the same pass, and its backward
// (mni_rocm_qk_norm_rope).  Bound by bandwidth where there are many rows: 8 bytes an element forward (one read, one
// write), 12 backward, and both run at the rate of a large copy (5.6 TB/s; less than the whole traffic need reach HBM):
// forward 5.8 TB/s on 2047 x 40 rows of 128 values (84 MB, 14.5 us), 6.3 on 8192 x 24 of 64 (101 MB, 16.0 us), backward
// 5.9 there (151 MB, 25.4 us).  A decoding step's 8 x 24 rows are one launch, 3.6 us.  All sums are fp32, the angles 64-bit.
#include <math.h>
#include <string.h>

#include "common.h"
#include "lanes.h"

namespace mni {
namespace {

constexpr int ROPE_TPB = 256;
constexpr int ROPE_MAX_DIM = 256;
constexpr int ROPE_BWD_GROUPS = 512;  // workgroups per operand in the backward: one partial sum of dgamma each

struct RopeArgs {
    mni_rope_heads q, k;
    const int32_t *positions;
    int64_t position_stride, offset;
    uint32_t tokens;
    float *part;  // backward: [2][ROPE_BWD_GROUPS][head_dim] partial sums of dgamma
    uint32_t seq, chunks;
    uint32_t first;  // forward: workgroups of the launches before
    int d, rot, interleaved;
    float eps, inv_d;
    double quarters[ROPE_MAX_DIM / 2];  // theta^(-2i / rot) / (pi / 2): quarter turns per position of pair i
};

// Eight values of a row per lane, as two pieces of four.  Rotated dims: with split halves lane l holds 4l .. 4l + 3 of
// either half, interleaved its first piece lies in the first half of the dims and its second in the second: either
// way a value and its partner sit in the same lane.  The lanes behind rot / 8 hold the unrotated dims, in order.
struct RopePlace {
    int lo, hi;   // first element of the two pieces
    bool live, turning;
};
__device__ __forceinline__ RopePlace rope_place(const RopeArgs &a, int l) {
    RopePlace p;
    p.turning = l < a.rot / 8;
    p.live = l < a.d / 8;
    if (p.turning) { p.lo = 4 * l; p.hi = a.rot / 2 + 4 * l; }
    else { p.lo = a.rot + 8 * (l - a.rot / 8); p.hi = p.lo + 4; }
    return p;
}
// cos and sin of at * f quarter turns.  In 64 bits, less whole quarter turns (1.5 * 2^52 added leaves the nearest whole number in
// the sum's last bits, whose last two are the quadrant); the rest, half a quarter turn at most, is rounded to 32 bits, which costs
// 0.4 * 2^-24, and goes through the Taylor polynomials of sin(pi r / 2) to r^9 and cos(pi r / 2) to r^10 (the next terms are
// below 2^-28).  Off by 1.4 * 2^-24 at most, and by three half steps of the result where that is small; the fraction of a whole
// turn rounded to 32 bits before sincospif was off by 1.8, by all bits next to a zero, and took 54.0 us where this takes 53.5 (8 x
// 1024 x 24 rows of 64, both ways).  Far positions add the frequency's rounding, 1.5 * 2^-53 of the angle.
__device__ __forceinline__ void rope_turn(double at, double f, float &c, float &s) {
    const double shift = 6755399441055744.0, moved = fma(at, f, shift);
    const uint32_t quadrant = (uint32_t)__double2loint(moved);
    const float r = (float)fma(at, f, shift - moved), z = r * r;
    const float tail = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.6044118e-4f, -4.6817541e-3f), 7.9692626e-2f), -6.4596410e-1f), -4.3711388e-8f);
    const float sine = fmaf(r, 1.57079637f, r * tail);  // (pi / 2 in two parts)
    const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.5202042e-5f, 9.1926027e-4f), -2.0863481e-2f), 2.5366951e-1f), -1.2337006f), 1.0f);
    const bool odd = quadrant & 1;
    s = __uint_as_float(__float_as_uint(odd ? cosine : sine) ^ ((quadrant & 2) << 30));
    c = __uint_as_float(__float_as_uint(odd ? sine : cosine) ^ (((quadrant + 1) & 2) << 30));
}
// cos and sin of the four pairs of a lane (pairs lo .. lo + 3; interleaved: lo / 2, lo / 2 + 1, hi / 2, hi / 2 + 1).
__device__ __forceinline__ void rope_angles(const RopeArgs &a, const double (&f)[4], uint32_t token, float (&c)[4], float (&s)[4]) {
    const uint32_t b = token / a.seq, t = token - b * a.seq;
    const double at = (double)((a.positions ? (int64_t)a.positions[b * a.position_stride + t] : (int64_t)t) + a.offset);
#pragma unroll
    for (int j = 0; j < 4; ++j) rope_turn(at, f[j], c[j], s[j]);
}
__device__ __forceinline__ void rope_quarters(const RopeArgs &a, const RopePlace &p, double (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int pair = a.interleaved ? (j < 2 ? p.lo / 2 + j : p.hi / 2 + j - 2) : p.lo + j;
        f[j] = p.turning ? a.quarters[pair] : 0.0;
    }
}
// (v0 .. v7) turned by +angle (SIGN 1) or -angle (SIGN -1)
template <int SIGN>
__device__ __forceinline__ void rope_rotate(bool interleaved, float (&v)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float &x = interleaved ? v[2 * j] : v[j], &y = interleaved ? v[2 * j + 1] : v[4 + j];
        const float sj = SIGN * s[j], x0 = x, y0 = y;
        x = x0 * c[j] - y0 * sj;
        y = y0 * c[j] + x0 * sj;
    }
}
__device__ __forceinline__ void rope_load(const float *row, const RopePlace &p, float (&v)[8]) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (p.live) {
        a = *reinterpret_cast<const float4 *>(row + p.lo);
        b = *reinterpret_cast<const float4 *>(row + p.hi);
    }
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void rope_store(float *row, const RopePlace &p, const float (&v)[8]) {
    if (!p.live) return;
    *reinterpret_cast<float4 *>(row + p.lo) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(row + p.hi) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ const float *rope_row(const mni_rope_heads &o, const RopeArgs &a, uint32_t token, int h) {
    const uint32_t b = token / a.seq, t = token - b * a.seq;
    return o.x + b * o.batch_stride + h * o.head_stride + t * o.token_stride;
}
__device__ __forceinline__ int64_t rope_out(const mni_rope_heads &o, const RopeArgs &a, uint32_t token, int h) {
    const uint32_t b = token / a.seq, t = token - b * a.seq;
    return (((int64_t)b * o.heads + h) * a.seq + t) * a.d;
}

// Forward.  LPR lanes hold a row; a group of LPR lanes takes the heads chunk, chunk + chunks, ... of one token (queries
// first, then keys), HPG of them: neighbouring groups read neighbouring heads, the sines are computed once for the HPG
// rows, and those are all asked for before.  (HPG is 4 from 65536 rows on, where there are groups enough for it; below, 1.)
template <int LPR, int HPG>
__global__ __launch_bounds__(ROPE_TPB) void rope_forward_kernel(const RopeArgs a) {
    const uint32_t item = (a.first + blockIdx.x) * (ROPE_TPB / LPR) + threadIdx.x / LPR;
    const uint32_t token = item / a.chunks;
    const int chunk = (int)(item - token * a.chunks);
    if (token >= a.tokens) return;  // (whole groups leave: nothing below crosses a group)
    const RopePlace p = rope_place(a, threadIdx.x % LPR);
    const int heads = (int)(a.q.heads + a.k.heads);
    double f[4];
    rope_quarters(a, p, f);
    float v[HPG][8];
#pragma unroll
    for (int j = 0; j < HPG; ++j) {
        const int h = chunk + j * a.chunks;
        const bool is_q = h < a.q.heads;
        if (h < heads) rope_load(is_q ? rope_row(a.q, a, token, h) : rope_row(a.k, a, token, h - (int)a.q.heads), p, v[j]);
    }
    float c[4], s[4];
    rope_angles(a, f, token, c, s);
#pragma unroll
    for (int j = 0; j < HPG; ++j) {
        const int h = chunk + j * a.chunks;
        if (h >= heads) break;
        const bool is_q = h < a.q.heads;
        float g[8], sum = 0.f;
        rope_load(is_q ? a.q.gamma : a.k.gamma, p, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += v[j][e] * v[j][e];
        const float r = rsqrtf(lanes_sum<LPR>(sum) * a.inv_d + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= r * g[e];
        if (p.turning) rope_rotate<1>(a.interleaved, v[j], c, s);
        rope_store(is_q ? a.q.out + rope_out(a.q, a, token, h) : a.k.out + rope_out(a.k, a, token, h - (int)a.q.heads), p, v[j]);
    }
}

// Backward of one operand (blockIdx.y: queries, keys).  A group of lanes takes row after row of (token, head), so that the
// sum for dgamma stays in registers: a workgroup leaves one partial row of it, 512 at most, which one more small launch
// adds up in order (2 us for few, 3.8 for 512; atomics would save it and make the bits a matter of chance).
template <int LPR>
__global__ __launch_bounds__(ROPE_TPB) void rope_backward_kernel(const RopeArgs a) {
    constexpr int GROUPS = ROPE_TPB / LPR;
    __shared__ float red[GROUPS][LPR * 8];
    const mni_rope_heads &o = blockIdx.y == 0 ? a.q : a.k;
    const int group = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const RopePlace p = rope_place(a, l);
    double f[4];
    rope_quarters(a, p, f);
    float g[8], acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    if (o.heads > 0 && o.grad) {
        rope_load(o.gamma, p, g);
        const uint32_t heads = (uint32_t)o.heads, rows = a.tokens * heads;
        for (uint32_t row = blockIdx.x * GROUPS + group; row < rows; row += gridDim.x * GROUPS) {
            const uint32_t token = row / heads;
            const int h = (int)(row - token * heads);
            float x[8], dz[8];
            rope_load(rope_row(o, a, token, h), p, x);
            const int64_t at = rope_out(o, a, token, h);
            rope_load(o.grad + at, p, dz);
            float c[4], s[4], sum = 0.f, dot = 0.f;
            rope_angles(a, f, token, c, s);
            if (p.turning) rope_rotate<-1>(a.interleaved, dz, c, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum += x[e] * x[e];
                dot += dz[e] * g[e] * x[e];
            }
            const float r = rsqrtf(lanes_sum<LPR>(sum) * a.inv_d + a.eps);
            const float k = lanes_sum<LPR>(dot) * a.inv_d * r * r * r;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                acc[e] += dz[e] * x[e] * r;
                dz[e] = dz[e] * g[e] * r - x[e] * k;
            }
            rope_store(o.dx + at, p, dz);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[group][l * 8 + e] = acc[e];
    __syncthreads();
    // one thread per dim: element e of lane l is dim lo + e (first piece) or hi + e - 4
    if (threadIdx.x < LPR * 8) {
        const int from = threadIdx.x / 8, e = threadIdx.x % 8;
        const RopePlace pl = rope_place(a, from);
        if (pl.live) {
            float sum = 0.f;
            for (int w = 0; w < GROUPS; ++w) sum += red[w][threadIdx.x];
            a.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.d + (e < 4 ? pl.lo + e : pl.hi + e - 4)] = sum;
        }
    }
}
// dgamma of both operands: 64 dims per workgroup, 16 wavefronts share the partial rows, added in wavefront order.
__global__ __launch_bounds__(1024) void rope_dgamma_kernel(const RopeArgs a, int rows) {
    __shared__ float red[16][64];
    const mni_rope_heads &o = blockIdx.y == 0 ? a.q : a.k;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = blockIdx.x * 64 + lane;
    float sum = 0.f;
    if (dim < a.d)
#pragma unroll 8
        for (int r = wave; r < rows; r += 16) sum += a.part[((int64_t)blockIdx.y * rows + r) * a.d + dim];
    red[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && dim < a.d && o.heads > 0 && o.grad) {
        for (int w = 1; w < 16; ++w) sum += red[w][lane];
        o.dgamma[dim] = sum;
    }
}

// Any head_dim, rotary_dims and alignment: a wavefront per row, a lane per pair and per unrotated value; 4-byte loads, and
// rows of few values leave lanes idle.
__device__ __forceinline__ void rope_pair(const RopeArgs &a, int i, int &lo, int &hi) {
    lo = a.interleaved ? 2 * i : i;
    hi = a.interleaved ? 2 * i + 1 : i + a.rot / 2;
}
__device__ __forceinline__ void rope_sincos(const RopeArgs &a, uint32_t token, int i, float &c, float &s) {
    const uint32_t b = token / a.seq, t = token - b * a.seq;
    rope_turn((double)((a.positions ? (int64_t)a.positions[b * a.position_stride + t] : (int64_t)t) + a.offset), a.quarters[i], c, s);
}
__global__ __launch_bounds__(ROPE_TPB) void rope_forward_any_kernel(const RopeArgs a) {
    const int heads = (int)(a.q.heads + a.k.heads), lane = threadIdx.x & 63;
    const uint32_t row = (a.first + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= a.tokens * heads) return;
    const uint32_t token = row / heads;
    int h = (int)(row - token * heads);
    const mni_rope_heads &o = h < a.q.heads ? a.q : a.k;
    if (h >= a.q.heads) h -= (int)a.q.heads;
    const float *x = rope_row(o, a, token, h);
    float *y = o.out + rope_out(o, a, token, h);
    float sum = 0.f;
    for (int e = lane; e < a.d; e += 64) sum += x[e] * x[e];
    const float r = rsqrtf(lanes_sum<64>(sum) * a.inv_d + a.eps);
    for (int i = lane; i < a.rot / 2; i += 64) {
        int lo, hi;
        rope_pair(a, i, lo, hi);
        float c, s;
        rope_sincos(a, token, i, c, s);
        const float zl = x[lo] * (r * o.gamma[lo]), zh = x[hi] * (r * o.gamma[hi]);
        y[lo] = zl * c - zh * s;
        y[hi] = zh * c + zl * s;
    }
    for (int e = a.rot + lane; e < a.d; e += 64) y[e] = x[e] * (r * o.gamma[e]);
}
__global__ __launch_bounds__(ROPE_TPB) void rope_backward_any_kernel(const RopeArgs a) {
    __shared__ float red[4][ROPE_MAX_DIM];
    const mni_rope_heads &o = blockIdx.y == 0 ? a.q : a.k;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int e = lane; e < a.d; e += 64) red[wave][e] = 0.f;  // dgamma of this wavefront
    __syncthreads();
    const uint32_t heads = (uint32_t)o.heads, rows = o.grad ? a.tokens * heads : 0;
    for (uint32_t row = blockIdx.x * 4 + wave; row < rows; row += gridDim.x * 4) {
        const uint32_t token = row / heads;
        const int h = (int)(row - token * heads);
        const float *x = rope_row(o, a, token, h);
        const int64_t at = rope_out(o, a, token, h);
        const float *dy = o.grad + at;
        float sum = 0.f, dot = 0.f;
        for (int i = lane; i < a.rot / 2; i += 64) {
            int lo, hi;
            rope_pair(a, i, lo, hi);
            float c, s;
            rope_sincos(a, token, i, c, s);
            sum += x[lo] * x[lo] + x[hi] * x[hi];
            dot += (dy[lo] * c + dy[hi] * s) * o.gamma[lo] * x[lo] + (dy[hi] * c - dy[lo] * s) * o.gamma[hi] * x[hi];
        }
        for (int e = a.rot + lane; e < a.d; e += 64) {
            sum += x[e] * x[e];
            dot += dy[e] * o.gamma[e] * x[e];
        }
        const float r = rsqrtf(lanes_sum<64>(sum) * a.inv_d + a.eps);
        const float k = lanes_sum<64>(dot) * a.inv_d * r * r * r;
        for (int i = lane; i < a.rot / 2; i += 64) {
            int lo, hi;
            rope_pair(a, i, lo, hi);
            float c, s;
            rope_sincos(a, token, i, c, s);
            const float zl = dy[lo] * c + dy[hi] * s, zh = dy[hi] * c - dy[lo] * s;
            red[wave][lo] += zl * x[lo] * r;
            red[wave][hi] += zh * x[hi] * r;
            o.dx[at + lo] = zl * o.gamma[lo] * r - x[lo] * k;
            o.dx[at + hi] = zh * o.gamma[hi] * r - x[hi] * k;
        }
        for (int e = a.rot + lane; e < a.d; e += 64) {
            red[wave][e] += dy[e] * x[e] * r;
            o.dx[at + e] = dy[e] * o.gamma[e] * r - x[e] * k;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.d; e += ROPE_TPB)
        a.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.d + e] = red[0][e] + red[1][e] + red[2][e] + red[3][e];
}

// 16-byte pieces of eight values: dims in eights, rows and strides on 16 bytes.
bool rope_in_pieces(const mni_rope_desc &d, bool backward) {
    if (d.head_dim % 8 || d.rotary_dims % 8) return false;
    for (const mni_rope_heads *o : {&d.q, &d.k}) {
        if (o->heads == 0 || (backward && !o->grad)) continue;
        const uintptr_t bits = (uintptr_t)o->x | (uintptr_t)o->gamma | (backward ? (uintptr_t)o->grad | (uintptr_t)o->dx : (uintptr_t)o->out);
        if (bits & 15) return false;
        if ((o->batch_stride | o->head_stride | o->token_stride) & 3) return false;
    }
    return true;
}
int rope_args(const mni_rope_desc &d, bool backward, RopeArgs *a) {
    const char *what = backward ? "qk_norm_rope_backward" : "qk_norm_rope";
    if (d.batch < 0 || d.seq < 0 || d.q.heads < 0 || d.k.heads < 0) return set_error(MNI_ERR_INVALID, "%s: negative extent", what);
    if (d.head_dim < 1 || d.head_dim > ROPE_MAX_DIM)
        return set_error(MNI_ERR_INVALID, "%s: head_dim %lld not in 1 .. %d", what, (long long)d.head_dim, ROPE_MAX_DIM);
    if (d.rotary_dims < 0 || d.rotary_dims > d.head_dim || d.rotary_dims % 2)
        return set_error(MNI_ERR_INVALID, "%s: rotary_dims %lld must be even and at most head_dim %lld", what, (long long)d.rotary_dims, (long long)d.head_dim);
    if (!(d.theta > 0.0) || !isfinite(d.theta)) return set_error(MNI_ERR_INVALID, "%s: theta must be positive", what);
    if (d.theta < 0x1p-16)  // (a position below 2^33 then stays below 2^49 quarter turns, which rope_turn takes apart; from 1 on, below 2^33)
        return set_error(MNI_ERR_INVALID, "%s: theta %g below 2^-16", what, d.theta);
    if (!(d.eps >= 0.0) || !isfinite(d.eps)) return set_error(MNI_ERR_INVALID, "%s: eps must not be negative", what);
    const int64_t far = (int64_t)1 << 32;
    if (d.offset < -far || d.offset > far)  // (the 64-bit angle loses its fraction on the way, and beside INT64_MAX the sum its sign)
        return set_error(MNI_ERR_INVALID, "%s: offset %lld beyond 2^32", what, (long long)d.offset);
    const int64_t most = (int64_t)1 << 31;
    if (d.seq > most || d.batch > most || d.q.heads > (1 << 20) || d.k.heads > (1 << 20) || (d.seq && d.batch > most / d.seq))
        return set_error(MNI_ERR_INVALID, "%s: more than 2^31 tokens or 2^20 heads", what);
    for (const mni_rope_heads *o : {&d.q, &d.k}) {
        if (o->heads == 0 || d.batch * d.seq == 0) continue;
        if (!o->x || !o->gamma || (!backward && !o->out) || (backward && o->grad && (!o->dx || !o->dgamma)))
            return set_error(MNI_ERR_INVALID, "%s: null operand", what);
    }
    a->q = d.q;
    a->k = d.k;
    a->positions = d.positions;
    a->position_stride = d.position_stride;
    a->offset = d.offset;
    // rows are counted in 32 bits, with room for the last workgroup's and the last round's overshoot
    if (d.batch * d.seq * (d.q.heads + d.k.heads) > ((int64_t)1 << 31))
        return set_error(MNI_ERR_INVALID, "%s: more than 2^31 rows", what);
    a->tokens = (uint32_t)(d.batch * d.seq);
    a->part = nullptr;
    a->seq = (uint32_t)(d.seq ? d.seq : 1);
    a->d = (int)d.head_dim;
    a->rot = (int)d.rotary_dims;
    a->interleaved = d.interleaved != 0;
    a->chunks = 1;
    a->first = 0;
    a->eps = (float)d.eps;
    a->inv_d = 1.0f / (float)d.head_dim;
    // The last plan's frequencies are kept: 64 powers take as long as a launch (calls that alternate between two plans pay that).
    static double quarters[ROPE_MAX_DIM / 2], of_theta = 0.0;
    static int of_rot = -1;
    if (of_theta != d.theta || of_rot != a->rot) {
        for (int i = 0; i < ROPE_MAX_DIM / 2; ++i) quarters[i] = i < a->rot / 2 ? pow(d.theta, -2.0 * i / a->rot) / M_PI_2 : 0.0;
        of_theta = d.theta;
        of_rot = a->rot;
    }
    memcpy(a->quarters, quarters, sizeof quarters);
    return MNI_OK;
}
// `blocks` workgroups, in as many launches as grids are needed for them.
template <class K>
void rope_launch(K kernel, RopeArgs &a, int64_t blocks) {
    for (int64_t first = 0; first < blocks; first += most_blocks(ROPE_TPB)) {
        a.first = (uint32_t)first;
        const int64_t some = blocks - first < most_blocks(ROPE_TPB) ? blocks - first : most_blocks(ROPE_TPB);
        MNI_KERNEL_LAUNCH(kernel, dim3((unsigned)some), dim3(ROPE_TPB), 0, ctx().stream, a);
    }
}
template <int LPR>
void rope_launch_forward(RopeArgs &a) {
    const int64_t heads = a.q.heads + a.k.heads;
    const int per_group = a.tokens * heads >= 65536 ? 4 : 1;
    a.chunks = (uint32_t)((heads + per_group - 1) / per_group);
    const int64_t blocks = ((int64_t)a.tokens * a.chunks + ROPE_TPB / LPR - 1) / (ROPE_TPB / LPR);
    if (per_group == 4) rope_launch(rope_forward_kernel<LPR, 4>, a, blocks);
    else rope_launch(rope_forward_kernel<LPR, 1>, a, blocks);
}

}  // namespace

int k_qk_norm_rope(const mni_rope_desc &d) {
    RopeArgs a;
    MNI_TRY(rope_args(d, false, &a));
    const int64_t rows = (int64_t)a.tokens * (d.q.heads + d.k.heads);
    if (rows == 0) return MNI_OK;
    MNI_TRY(ensure_init());
    if (!rope_in_pieces(d, false)) rope_launch(rope_forward_any_kernel, a, (rows + 3) / 4);
    else if (a.d <= 32) rope_launch_forward<4>(a);
    else if (a.d <= 64) rope_launch_forward<8>(a);
    else if (a.d <= 128) rope_launch_forward<16>(a);
    else rope_launch_forward<32>(a);
    return check_launch("qk_norm_rope");
}

int k_qk_norm_rope_backward(const mni_rope_desc &d) {
    RopeArgs a;
    MNI_TRY(rope_args(d, true, &a));
    MNI_TRY(ensure_init());
    bool any = false;  // rows that a gradient comes from
    for (const mni_rope_heads *o : {&d.q, &d.k}) {
        if (!o->grad) continue;
        if (a.tokens > 0 && o->heads > 0) any = true;
        else if (o->dgamma) MNI_TRY(k_fill(o->dgamma, 0.0f, a.d));  // a sum over no rows
    }
    if (!any) return MNI_OK;
    const int64_t heads = d.q.heads > d.k.heads ? d.q.heads : d.k.heads;
    const bool pieces = rope_in_pieces(d, true);
    const int lpr = !pieces ? 64 : a.d <= 32 ? 4 : a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32;
    int64_t blocks = ((int64_t)a.tokens * heads + ROPE_TPB / lpr - 1) / (ROPE_TPB / lpr);
    if (blocks > ROPE_BWD_GROUPS) blocks = ROPE_BWD_GROUPS;
    void *part = nullptr;
    MNI_TRY(dev_alloc(&part, (size_t)(2 * blocks * a.d) * sizeof(float)));
    a.part = (float *)part;
    const dim3 grid((unsigned)blocks, 2), block(ROPE_TPB);
    hipStream_t st = ctx().stream;
    if (!pieces) MNI_KERNEL_LAUNCH(rope_backward_any_kernel, grid, block, 0, st, a);
    else if (lpr == 4) MNI_KERNEL_LAUNCH((rope_backward_kernel<4>), grid, block, 0, st, a);
    else if (lpr == 8) MNI_KERNEL_LAUNCH((rope_backward_kernel<8>), grid, block, 0, st, a);
    else if (lpr == 16) MNI_KERNEL_LAUNCH((rope_backward_kernel<16>), grid, block, 0, st, a);
    else MNI_KERNEL_LAUNCH((rope_backward_kernel<32>), grid, block, 0, st, a);
    int rc = check_launch("qk_norm_rope_backward");
    if (rc == MNI_OK) {
        MNI_KERNEL_LAUNCH(rope_dgamma_kernel, dim3((unsigned)((a.d + 63) / 64), 2), dim3(1024), 0, st, a, (int)blocks);
        rc = check_launch("qk_norm_rope_backward");
    }
    dev_free(part);
    return rc;
}

}  // namespace mni

extern "C" {

int mni_rocm_qk_norm_rope(const mni_rope_desc *desc) {
    MNI_API_GUARD;
    if (!desc) return mni::set_error(MNI_ERR_INVALID, "qk_norm_rope: null descriptor");
    return mni::k_qk_norm_rope(*desc);
}
int mni_rocm_qk_norm_rope_backward(const mni_rope_desc *desc) {
    MNI_API_GUARD;
    if (!desc) return mni::set_error(MNI_ERR_INVALID, "qk_norm_rope_backward: null descriptor");
    return mni::k_qk_norm_rope_backward(*desc);
}

}  // extern "C"
