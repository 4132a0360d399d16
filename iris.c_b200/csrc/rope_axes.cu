/*
 * Rotation from token positions with several axes (time, height, width, ...),
 * as tables and inside the Q/K norm.
 *
 * Pair j of a head turns by p[s, axis(j)] * f_j. f_j / 2 pi is kept as a
 * 64-bit fraction of a turn F_j, so the phase of a row is p * F_j modulo 2^64:
 * whole turns fall off by themselves, for any sign and size of p; there is no
 * range reduction and no table. The fraction is cut, not rounded, and comes from
 * a frequency in long double, so the phase is off by up to |p| 2^-64 (1 + r f_j /
 * 2 pi) turns with r = 5 roundings and the logarithm of the power of theta, 19 at
 * most for theta 1e6: at |p| 2^31 and f_j 1 that is 4.7e-10 turns (2.9e-9 rad). Of the
 * phase the top 32 bits are used (2^-32 turns = 1.5e-9 rad): the two highest
 * give the quadrant after rounding, the rest an angle a within pi / 4 on which
 * a + a^3 S(a^2) and 1 - a^2 / 2 + a^4 C(a^2), with quadratics S and C of least
 * maximum error (an iteratively reweighted least-squares fit), are within
 * 2.3e-9 of sine and cosine, below the rounding of fp32.
 *
 * k_rope_tables writes 8 bytes per pair and is bound by those stores: 134 866
 * rows of 64 pairs (71 MB) take 13.4 us, 5.3 TB/s, of which a fill of the same
 * bytes takes 10.4; a thread keeps its pairs and walks the rows, so that the
 * plan is read once.
 *
 * k_qk_norm_rope_axes reads and writes every element once and is bound by
 * HBM. LANES = head_dim / 8 lanes own one (row, head) unit, 16 bytes each. A
 * lane holds both members of its four pairs 4 l .. 4 l + 3 in either pairing
 * (one 16-byte access, or two of 8 bytes half a head apart), so the rotation
 * needs no exchange. A warp takes one row and a run of its heads: its lanes
 * work out the head_dim / 2 sines and cosines of the row together, hand each
 * other the four they need by shuffles, and fold them with the norm weights
 * once per row. 16 896 rows x 64 heads (554 MB) take 91 us, 6.1 TB/s; split
 * halves without a norm, 31 005 x 36 heads (572 MB), 92 us, 6.2 TB/s; 768 x 60
 * heads 7.8 us, launch and one wave of loads.
 */
#include "common.cuh"

#include <math.h>

#include "iris_dev.h"

namespace iris_b200 {
namespace rope_axes {

static constexpr int kThreads = 256;
static constexpr int kBlocksPerSM = 4;       /* of k_rope_tables */
static constexpr int kTableRows = 4;         /* rows of a thread of k_rope_tables whose positions are in flight */
static constexpr int kMaxPairs = IRIS_B200_ROPE_MAX_PAIRS;

/* F_j as two words of which the lower counts as signed: F_j = hi 2^32 + lo modulo 2^64. */
struct Turn {
    uint32_t hi;
    int lo;
};
struct Plan {
    int n;                                   /* positions per row */
    Turn turn[kMaxPairs];
    unsigned char axis[kMaxPairs];
};

/* An address inside the launch's parameters as a plain one: lanes that read
 * different entries through the constant cache would be served one after the
 * other (768 x 60 heads: 11.0 us so, 9.1 us through loads). */
template <typename T>
__device__ __forceinline__ const T *plain(const T *param) {
    asm("" : "+l"(param));
    return param;
}

/* cos and sin of the phase p * turn. */
__device__ __forceinline__ void turn_of(int p, Turn t, float &cs, float &sn) {
    /* Bits 32 to 63 of the phase plus an eighth of a turn: two bits of quadrant, then the angle from -pi / 4 up. */
    const uint32_t top = (uint32_t)p * t.hi + (uint32_t)__mulhi(p, t.lo) + 0x20000000u;
    const float a = (float)((int)(top & 0x3FFFFFFFu) - 0x20000000) * 1.4629180792671596e-09f;     /* 2 pi / 2^32 */
    const float b = a * a;
    float s = fmaf(b, -0.00019495636f, 0.008331979f);
    s = fmaf(b, s, -0.16666651f);
    s = fmaf(a * b, s, a);
    float c = fmaf(b, 2.4438452e-05f, -0.0013887368f);
    c = fmaf(b, c, 0.041666646f);
    c = fmaf(b, c, -0.5f);
    c = fmaf(b, c, 1.0f);
    const bool odd = top & 0x40000000u;
    const float x = odd ? s : c, y = odd ? c : s;
    /* cos: + - - + over the quadrants, sin: + + - -. */
    cs = __uint_as_float(__float_as_uint(x) ^ ((top + 0x40000000u) & 0x80000000u));
    sn = __uint_as_float(__float_as_uint(y) ^ (top & 0x80000000u));
}

/* Both 16-byte kernels start under the kernel ahead of them and wait for its
 * end. What they read may be written until then, so it is never read through
 * the non-coherent path, which takes memory as constant for the whole kernel:
 * no __ldg and no __restrict__ here. */

/* ---- tables ---- */

/* A thread keeps VEC consecutive pairs for all its rows. */
template <int VEC>
__global__ void __launch_bounds__(kThreads, kBlocksPerSM)
k_rope_tables(float *cos_out, float *sin_out, const int *pos, int seq, int half,
              const __grid_constant__ Plan plan) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int per_row = half / VEC, rows_per_block = kThreads / per_row;
    const int r = threadIdx.x / per_row, j = (threadIdx.x - r * per_row) * VEC;
    if (r >= rows_per_block) return;
    Turn turn[VEC];
    int axis[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        turn[i] = plain(plan.turn)[j + i];
        axis[i] = plain(plan.axis)[j + i];
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long stride = (long long)gridDim.x * rows_per_block;
    for (long long row0 = (long long)blockIdx.x * rows_per_block + r; row0 < seq; row0 += kTableRows * stride) {
        int at[kTableRows][VEC];
#pragma unroll
        for (int k = 0; k < kTableRows; k++) {
            const long long row = row0 + k * stride < seq ? row0 + k * stride : row0;
            const int *p = pos + row * plan.n;
            /* Neighbouring pairs mostly belong to one axis. */
#pragma unroll
            for (int i = 0; i < VEC; i++) at[k][i] = i > 0 && axis[i] == axis[i > 0 ? i - 1 : 0] ? at[k][i > 0 ? i - 1 : 0] : p[axis[i]];
        }
#pragma unroll
        for (int k = 0; k < kTableRows; k++) {
            const long long row = row0 + k * stride;
            if (row >= seq) break;
            float c[VEC], s[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) turn_of(at[k][i], turn[i], c[i], s[i]);
            float *co = cos_out + row * half + j, *so = sin_out + row * half + j;
            if (VEC == 4) {
                __stcs(reinterpret_cast<float4 *>(co), make_float4(c[0], c[1 % VEC], c[2 % VEC], c[3 % VEC]));
                __stcs(reinterpret_cast<float4 *>(so), make_float4(s[0], s[1 % VEC], s[2 % VEC], s[3 % VEC]));
            } else {
                *co = c[0];
                *so = s[0];
            }
        }
    }
}

/* ---- norm and rotation ---- */

struct Rows {
    uint16_t *out[2];           /* Q, K */
    const uint16_t *in[2];
    const float *w[2];
    int ldo[2];
    int ldi;
    int heads[2];
    const int *pos;
    int seq;
    int chunk, chunks;          /* heads of a row per warp, warps per row */
    float eps;
};

/* Units of a lane group that are loaded before the first is used, and CTAs per
 * SM. The 8-byte accesses of the split pairing want twice as many in flight. At
 * 16 896 x 64 heads (554 MB) without the split: 4 units and 3 CTAs 94 us, 4 and
 * 4 107, 8 and 2 96, 6 and 3 95, 2 and 6 125. With it, at 31 005 x 36 heads (572
 * MB): 8 and 2 94 us, 4 and 3 102, 8 and 3 103. */
template <bool SPLIT>
struct Shape {
    static constexpr int kInFlight = SPLIT ? 8 : 4;
    static constexpr int kBlocks = SPLIT ? 2 : 3;
};

template <int HD, bool SPLIT, bool NORM>
__global__ void __launch_bounds__(kThreads, Shape<SPLIT>::kBlocks)
k_qk_norm_rope_axes(const __grid_constant__ Rows a, const __grid_constant__ Plan plan) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int LANES = HD / 8;                   /* lanes of a unit */
    constexpr int GROUPS = 32 / LANES;              /* units a warp works on at a time */
    constexpr int PPL = HD / 64;                    /* pairs whose sine and cosine a lane works out */
    constexpr int FLIGHT = Shape<SPLIT>::kInFlight;
    const int lane = threadIdx.x & 31, l = lane & (LANES - 1), grp = lane / LANES;
    /* The lane's pairs 4 l .. 4 l + 3 in memory. */
    const int d0 = SPLIT ? 4 * l : 8 * l, d1 = SPLIT ? HD / 2 + 4 * l : 8 * l + 4;
    Turn turn[PPL];
    int axis[PPL];
#pragma unroll
    for (int i = 0; i < PPL; i++) {
        turn[i] = plain(plan.turn)[lane * PPL + i];
        axis[i] = plain(plan.axis)[lane * PPL + i];
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long items = (long long)a.seq * a.chunks;
    const long long warps = (long long)gridDim.x * (kThreads / 32);
    for (long long item = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += warps) {
        const int row = (int)(item / a.chunks);
        const int u0 = (int)(item - (long long)row * a.chunks) * a.chunk;     /* first head, Q heads before K heads */
        const int u1 = u0 + a.chunk;
        int part = u0 < a.heads[0] ? 0 : 1;
        int h = part ? u0 - a.heads[0] : u0;
        int h1 = part ? u1 - a.heads[0] : u1;
        if (h1 > a.heads[part]) h1 = a.heads[part];
        uint2 va[FLIGHT], vb[FLIGHT];
        auto load = [&]() {
            const uint16_t *in = a.in[part] + (size_t)row * a.ldi;
#pragma unroll
            for (int i = 0; i < FLIGHT; i++) {
                const int hh = h + i * GROUPS + grp;
                va[i] = vb[i] = make_uint2(0u, 0u);
                if (hh < h1) {
                    const uint16_t *src = in + hh * HD;
                    if (SPLIT) {
                        va[i] = *reinterpret_cast<const uint2 *>(src + d0);
                        vb[i] = *reinterpret_cast<const uint2 *>(src + d1);
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4 *>(src + d0);
                        va[i] = make_uint2(v.x, v.y);
                        vb[i] = make_uint2(v.z, v.w);
                    }
                }
            }
        };
        load();                         /* under the way to the row's angles */
        float cs[4], sn[4];
        {
            float c[PPL], s[PPL];
#pragma unroll
            for (int i = 0; i < PPL; i++) turn_of(a.pos[(size_t)row * plan.n + axis[i]], turn[i], c[i], s[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int src = (4 * l + i) / PPL;
                cs[i] = __shfl_sync(0xffffffffu, c[i % PPL], src);
                sn[i] = __shfl_sync(0xffffffffu, s[i % PPL], src);
            }
        }
        for (;;) {
            /* Pair i of the lane is (x[i], x[4 + i]) with SPLIT, (x[2 i], x[2 i + 1]) without. */
            float k00[4], k01[4], k10[4], k11[4];
            if (NORM) {
                const float4 w0 = *reinterpret_cast<const float4 *>(a.w[part] + d0);
                const float4 w1 = *reinterpret_cast<const float4 *>(a.w[part] + d1);
                const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float wa = w[SPLIT ? i : 2 * i], wb = w[SPLIT ? 4 + i : 2 * i + 1];
                    k00[i] = cs[i] * wa;
                    k01[i] = sn[i] * wb;
                    k10[i] = cs[i] * wb;
                    k11[i] = sn[i] * wa;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    k00[i] = k10[i] = cs[i];
                    k01[i] = k11[i] = sn[i];
                }
            }
            uint16_t *out = a.out[part] + (size_t)row * a.ldo[part];
            for (;;) {
#pragma unroll
                for (int i = 0; i < FLIGHT; i++) {
                    const int hh = h + i * GROUPS + grp;
                    float x[8] = {bf_lo(va[i].x), bf_hi(va[i].x), bf_lo(va[i].y), bf_hi(va[i].y),
                                  bf_lo(vb[i].x), bf_hi(vb[i].x), bf_lo(vb[i].y), bf_hi(vb[i].y)};
                    float inv = 1.0f;
                    if (NORM) {
                        float ss = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; j++) ss = fmaf(x[j], x[j], ss);
#pragma unroll
                        for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                        inv = rsqrtf(ss * (1.0f / HD) + a.eps);
                    }
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int ia = SPLIT ? j : 2 * j, ib = SPLIT ? 4 + j : 2 * j + 1;
                        y[ia] = (x[ia] * k00[j] - x[ib] * k01[j]) * inv;
                        y[ib] = (x[ib] * k10[j] + x[ia] * k11[j]) * inv;
                    }
                    if (hh < h1) {
                        uint16_t *dst = out + hh * HD;
                        const uint2 oa = make_uint2(cvt_bf16x2(y[0], y[1]), cvt_bf16x2(y[2], y[3]));
                        const uint2 ob = make_uint2(cvt_bf16x2(y[4], y[5]), cvt_bf16x2(y[6], y[7]));
                        if (SPLIT) {
                            *reinterpret_cast<uint2 *>(dst + d0) = oa;
                            *reinterpret_cast<uint2 *>(dst + d1) = ob;
                        } else {
                            *reinterpret_cast<uint4 *>(dst + d0) = make_uint4(oa.x, oa.y, ob.x, ob.y);
                        }
                    }
                }
                h += FLIGHT * GROUPS;
                if (h >= h1) break;
                load();
            }
            /* The K heads of the chunk, when it began among the Q heads. */
            if (part || u1 <= a.heads[0] || a.heads[1] == 0) break;
            part = 1;
            h = 0;
            h1 = u1 - a.heads[0] < a.heads[1] ? u1 - a.heads[0] : a.heads[1];
            load();
        }
    }
}

/* Any even head_dim up to 512, any alignment: one warp per (row, head), 2-byte
 * accesses, every unit works out its own angles. */
__global__ void __launch_bounds__(kThreads)
k_qk_norm_rope_axes_any(const __grid_constant__ Rows a, const __grid_constant__ Plan plan, int head_dim, int split_half) {
    const int lane = threadIdx.x & 31, half = head_dim / 2, per_row = a.heads[0] + a.heads[1];
    const long long units = (long long)a.seq * per_row;
    const long long warps = (long long)gridDim.x * (kThreads / 32);
    for (long long unit = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); unit < units; unit += warps) {
        const int row = (int)(unit / per_row), u = (int)(unit - (long long)row * per_row);
        const int part = u >= a.heads[0], h = part ? u - a.heads[0] : u;
        const uint16_t *in = a.in[part] + (size_t)row * a.ldi + (size_t)h * head_dim;
        uint16_t *out = a.out[part] + (size_t)row * a.ldo[part] + (size_t)h * head_dim;
        const float *w = a.w[part];
        float inv = 1.0f;
        if (w) {
            float ss = 0.0f;
            for (int d = lane; d < head_dim; d += 32) {
                const float x = bf2f(in[d]);
                ss = fmaf(x, x, ss);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(ss / head_dim + a.eps);
        }
        for (int j = lane; j < half; j += 32) {
            const int i0 = split_half ? j : 2 * j, i1 = split_half ? j + half : 2 * j + 1;
            float cs, sn;
            turn_of(a.pos[(size_t)row * plan.n + plain(plan.axis)[j]], plain(plan.turn)[j], cs, sn);
            const float x0 = bf2f(in[i0]) * (w ? inv * w[i0] : 1.0f), x1 = bf2f(in[i1]) * (w ? inv * w[i1] : 1.0f);
            out[i0] = (uint16_t)cvt_bf16x2(x0 * cs - x1 * sn, 0.0f);
            out[i1] = (uint16_t)cvt_bf16x2(x1 * cs + x0 * sn, 0.0f);
        }
    }
}

static int bad(const char *op, const char *why) {
    set_error(IRIS_B200_EINVAL, op, why);
    return IRIS_B200_EINVAL;
}

/* The caller's plan, checked again: it lives in the caller's memory. */
static bool plan_of(const iris_b200_rope_axes *axes, int head_dim, Plan *plan) {
    if (!axes || head_dim <= 0 || (head_dim & 1) || head_dim / 2 > kMaxPairs || axes->head_dim != head_dim || axes->n < 1 ||
        axes->n > IRIS_B200_ROPE_MAX_AXES)
        return false;
    plan->n = axes->n;
    for (int j = 0; j < head_dim / 2; j++) {
        if (axes->axis[j] >= axes->n) return false;
        const uint32_t lo = (uint32_t)axes->turn[j];
        plan->turn[j].hi = (uint32_t)(axes->turn[j] >> 32) + (lo >> 31);
        plan->turn[j].lo = (int)lo;
        plan->axis[j] = axes->axis[j];
    }
    return true;
}

static bool aligned(const void *p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

template <int HD>
static cudaError_t launch_rows(const cudaLaunchConfig_t &cfg, const Rows &a, const Plan &plan, bool split, bool norm) {
    if (split)
        return norm ? cudaLaunchKernelEx(&cfg, k_qk_norm_rope_axes<HD, true, true>, a, plan)
                    : cudaLaunchKernelEx(&cfg, k_qk_norm_rope_axes<HD, true, false>, a, plan);
    return norm ? cudaLaunchKernelEx(&cfg, k_qk_norm_rope_axes<HD, false, true>, a, plan)
                : cudaLaunchKernelEx(&cfg, k_qk_norm_rope_axes<HD, false, false>, a, plan);
}

/* Launch with programmatic stream serialisation (the kernels wait for the
 * grid ahead before they touch memory that it may have written). */
struct Launch {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    Launch(unsigned blocks) : cfg(), attr() {
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = g.stream;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
};

}  // namespace rope_axes
}  // namespace iris_b200

using namespace iris_b200;
using namespace iris_b200::rope_axes;

extern "C" int iris_b200_rope_axes_plan(iris_b200_rope_axes *axes, const int *dim, const double *scale, int n, double theta,
                                        int one_progression, int head_dim) {
    const char *op = "rope_axes_plan";
    if (!axes || !dim || n < 1 || n > IRIS_B200_ROPE_MAX_AXES || head_dim <= 0 || (head_dim & 1) || head_dim / 2 > kMaxPairs)
        return bad(op, "bad argument");
    if (!(theta > 0.0) || !isfinite(theta)) return bad(op, "theta must be positive");
    long long sum = 0;
    for (int a = 0; a < n; a++) {
        if (dim[a] < 0 || (dim[a] & 1)) return bad(op, "an axis turns an even number of dimensions");
        if (scale && !isfinite(scale[a])) return bad(op, "scales must be finite");
        sum += dim[a];
    }
    if (sum > head_dim) return bad(op, "the axes turn more dimensions than a head has");
    axes->n = n;
    axes->head_dim = head_dim;
    int j = 0;
    for (int a = 0; a < n; a++)
        for (int i = 0; i < dim[a] / 2; i++, j++) {
            const long double power = one_progression ? 2.0L * j / head_dim : 2.0L * i / dim[a];
            const long double turns = (long double)(scale ? scale[a] : 1.0) * powl((long double)theta, -power) /
                                      6.283185307179586476925286766559L;
            long double frac = turns - floorl(turns);
            if (!(frac >= 0.0L) || frac >= 1.0L) frac = 0.0L;
            axes->turn[j] = (uint64_t)(frac * 18446744073709551616.0L);
            axes->axis[j] = (uint8_t)a;
        }
    for (; j < IRIS_B200_ROPE_MAX_PAIRS; j++) {
        axes->turn[j] = 0;
        axes->axis[j] = 0;
    }
    return IRIS_B200_OK;
}

extern "C" int iris_b200_rope_axes_tables(float *cos_out, float *sin_out, const int *pos, const iris_b200_rope_axes *axes,
                                          int seq, int head_dim) {
    const char *op = "rope_axes_tables";
    Plan plan;
    if (seq < 0 || !plan_of(axes, head_dim, &plan)) return bad(op, "bad argument");
    if (seq > 0 && (!cos_out || !sin_out || !pos)) return bad(op, "bad argument");
    if (!require_device(op)) return IRIS_B200_ENODEV;
    if (seq == 0) return IRIS_B200_OK;
    const int half = head_dim / 2;
    const bool vec = half % 4 == 0 && aligned(cos_out, 16) && aligned(sin_out, 16);
    const int rows_per_block = kThreads / (vec ? half / 4 : half);
    long long blocks = ((long long)seq + rows_per_block - 1) / rows_per_block;
    if (blocks > (long long)g.sm_count * kBlocksPerSM) blocks = (long long)g.sm_count * kBlocksPerSM;
    Launch l((unsigned)blocks);
    const cudaError_t err = vec ? cudaLaunchKernelEx(&l.cfg, k_rope_tables<4>, cos_out, sin_out, pos, seq, half, plan)
                                : cudaLaunchKernelEx(&l.cfg, k_rope_tables<1>, cos_out, sin_out, pos, seq, half, plan);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}

extern "C" int iris_b200_qk_norm_rope_axes(uint16_t *q_out, int ldqo, uint16_t *k_out, int ldko, const uint16_t *q,
                                           const uint16_t *k, int ldi, const float *wq, const float *wk, const int *pos,
                                           const iris_b200_rope_axes *axes, int seq, int heads, int kv_heads, int head_dim,
                                           float eps, int split_half) {
    const char *op = "qk_norm_rope_axes";
    Plan plan;
    if (seq < 0 || heads <= 0 || kv_heads < 0 || !plan_of(axes, head_dim, &plan)) return bad(op, "bad argument");
    const bool has_k = kv_heads > 0;
    if ((long long)heads * head_dim > ldi || (long long)kv_heads * head_dim > ldi || (long long)heads * head_dim > ldqo ||
        (has_k && (long long)kv_heads * head_dim > ldko))
        return bad(op, "a row stride is shorter than a row of heads");
    if ((wq != NULL) != (wk != NULL) && has_k) return bad(op, "norm weights for one of Q and K only");
    if (!(eps >= 0.0f)) return bad(op, "eps must not be negative");
    if (seq > 0 && (!q_out || !q || !pos || (has_k && (!k_out || !k)))) return bad(op, "bad argument");
    /* In place means the same rows; anything else that overlaps would be read after it is written. */
    if (seq > 0 && ((q_out == q && ldqo != ldi) || (has_k && k_out == k && ldko != ldi)))
        return bad(op, "in place needs equal row strides");
    if (!require_device(op)) return IRIS_B200_ENODEV;
    if (seq == 0) return IRIS_B200_OK;
    Rows a = {};
    a.out[0] = q_out;
    a.in[0] = q;
    a.w[0] = wq;
    a.ldo[0] = ldqo;
    a.heads[0] = heads;
    if (has_k) {
        a.out[1] = k_out;
        a.in[1] = k;
        a.w[1] = wk;
        a.ldo[1] = ldko;
        a.heads[1] = kv_heads;
    }
    a.ldi = ldi;
    a.pos = pos;
    a.seq = seq;
    a.eps = eps;
    const int per_row = heads + kv_heads;
    const bool fast = (head_dim == 64 || head_dim == 128 || head_dim == 256) && ldi % 8 == 0 && ldqo % 8 == 0 &&
                      aligned(q, 16) && aligned(q_out, 16) && (!wq || aligned(wq, 16)) &&
                      (!has_k || (ldko % 8 == 0 && aligned(k, 16) && aligned(k_out, 16) && (!wk || aligned(wk, 16))));
    if (!fast) {
        long long blocks = ((long long)seq * per_row + kThreads / 32 - 1) / (kThreads / 32);
        if (blocks > (long long)g.sm_count * 32) blocks = (long long)g.sm_count * 32;
        k_qk_norm_rope_axes_any<<<(unsigned)blocks, kThreads, 0, g.stream>>>(a, plan, head_dim, split_half);
        return after_launch(op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
    }
    /* A row is cut into as many warps as it takes to fill the device once, in
     * pieces of whole batches (768 x 60 heads: 16 heads per warp 7.8 us, 12 heads
     * 9.1, 20 heads 8.8). */
    const int per_sm = split_half ? Shape<true>::kBlocks : Shape<false>::kBlocks;
    const long long slots = (long long)g.sm_count * per_sm * (kThreads / 32);
    const int batch = (split_half ? Shape<true>::kInFlight : Shape<false>::kInFlight) * (32 / (head_dim / 8));
    const long long chunks = (slots + seq - 1) / seq;
    a.chunk = (int)((per_row + chunks - 1) / chunks);
    a.chunk = (a.chunk + batch - 1) / batch * batch;
    a.chunks = (per_row + a.chunk - 1) / a.chunk;
    long long blocks = ((long long)seq * a.chunks + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > (long long)g.sm_count * per_sm) blocks = (long long)g.sm_count * per_sm;
    Launch l((unsigned)blocks);
    const bool split = split_half != 0, norm = wq != NULL;
    const cudaError_t err = head_dim == 64    ? launch_rows<64>(l.cfg, a, plan, split, norm)
                            : head_dim == 128 ? launch_rows<128>(l.cfg, a, plan, split, norm)
                                              : launch_rows<256>(l.cfg, a, plan, split, norm);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}
