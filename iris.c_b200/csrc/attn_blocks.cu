/*
 * Attention over lists of key blocks: argument checks, kernel choice, and the
 * general CUDA-core kernel.
 *
 * k_attention_blocks_any covers every argument domain (any head_dim up to
 * 512, any alignment, any block sizes). A CTA owns up to eight consecutive
 * queries of one head inside one query block, one warp per query; keys of the
 * listed blocks are staged in shared memory 32 at a time, each lane scores one
 * key, and the softmax runs with a running maximum and sum in fp32; the
 * probabilities meet V in fp32 too, as in the kernel for rows with a list of
 * their own (only the tensor cores want them as bf16). Rows of masked keys are
 * staged as zeros, so whatever they hold never meets a zero probability. It is
 * the form the tensor-core kernel is checked against.
 *
 * The automatic choice: rows with a list of their own go to the kernel that
 * reads keys into registers (attn_blocks_row.cu: 1 row 14.7 us against 19.1 on
 * the tensor cores, 256 rows 712 against 893), everything else that the
 * tensor-core kernel takes to that one, the rest to the general one.
 */
#include "common.cuh"

#include <limits.h>
#include <math.h>

#include "iris_dev.h"
#include "kernels.h"

namespace iris_b200 {

static constexpr int kQPerBlock = 8;
static constexpr int kKeysPerTile = 32;
static constexpr int kMaxHeadDim = 512;

__global__ void __launch_bounds__(kQPerBlock * 32)
k_attention_blocks_any(const BlockAttnArgs a, int tiles_per_block) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int hd = a.head_dim, kstride = hd + 2;      /* odd word stride: no bank conflicts */
    uint16_t *ks = reinterpret_cast<uint16_t *>(smem_raw);
    uint16_t *vs = ks + kKeysPerTile * kstride;
    float *qs = reinterpret_cast<float *>(vs + kKeysPerTile * hd);
    __shared__ unsigned usable;                       /* keys of the tile that count */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, kvh = h / (a.heads / a.kv_heads);
    const int qb = blockIdx.x / tiles_per_block;
    const int in_block = (blockIdx.x - qb * tiles_per_block) * kQPerBlock + warp;
    const long long qi = (long long)qb * a.q_block + in_block;
    const bool qvalid = in_block < a.q_block && qi < a.seq_q;
    const int ndim = (hd + 31) / 32;
    const float scale_log2 = a.scale * 1.4426950408889634f;

    float *qrow = qs + warp * hd;
    for (int d = lane; d < hd; d += 32) qrow[d] = qvalid ? bf2f(a.q[(size_t)qi * a.ldq + (size_t)h * hd + d]) : 0.0f;

    float acc[kMaxHeadDim / 32];
#pragma unroll
    for (int t = 0; t < kMaxHeadDim / 32; t++) acc[t] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int *list = a.list + ((size_t)h * a.q_blocks + qb) * a.list_len;

    for (int e = 0; e < a.list_len; e++) {
        const int b = list[e];
        if (b < 0 || b >= a.k_blocks) continue;
        const long long first = (long long)b * a.k_block;
        const int rows = (int)(a.seq_k - first < a.k_block ? a.seq_k - first : a.k_block);
        /* (64 bits: k0 passes the last row by more than a 31-bit count has room for.) */
        for (long long k0 = 0; k0 < rows; k0 += kKeysPerTile) {
            __syncthreads();
            if (warp == 0) {
                const bool ok = k0 + lane < rows && (!a.key_mask || a.key_mask[first + k0 + lane] != 0);
                const unsigned bits = __ballot_sync(0xffffffffu, ok);
                if (lane == 0) usable = bits;
            }
            __syncthreads();
            const unsigned bits = usable;
            for (int i = threadIdx.x; i < kKeysPerTile * hd; i += blockDim.x) {
                const int r = i / hd, d = i - r * hd;
                const bool ok = (bits >> r) & 1u;
                const size_t row = (size_t)(first + k0 + r), col = (size_t)kvh * hd + d;
                ks[r * kstride + d] = ok ? a.k[row * a.ldk + col] : (uint16_t)0;
                vs[r * hd + d] = ok ? a.v[row * a.ldv + col] : (uint16_t)0;
            }
            __syncthreads();
            float dot = 0.0f;
            const uint16_t *kr = ks + lane * kstride;
            for (int d = 0; d < hd; d++) dot = fmaf(qrow[d], bf2f(kr[d]), dot);
            const float sc = (bits >> lane) & 1u ? dot * scale_log2 : -INFINITY;
            float mx = sc;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mnew = fmaxf(m, mx);
            const float mref = mnew == -INFINITY ? 0.0f : mnew;
            const float alpha = exp2f(m - mref), p = exp2f(sc - mref);
            float ps = p;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
            l = l * alpha + ps;
            m = mnew;
#pragma unroll
            for (int t = 0; t < kMaxHeadDim / 32; t++) acc[t] *= alpha;
            for (int j = 0; j < kKeysPerTile; j++) {
                const float pj = __shfl_sync(0xffffffffu, p, j);
                const uint16_t *vr = vs + j * hd;
#pragma unroll
                for (int t = 0; t < kMaxHeadDim / 32; t++) {
                    const int d = lane + 32 * t;
                    if (t < ndim && d < hd) acc[t] = fmaf(pj, bf2f(vr[d]), acc[t]);
                }
            }
        }
    }
    if (!qvalid) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int t = 0; t < kMaxHeadDim / 32; t++) {
        const int d = lane + 32 * t;
        if (t < ndim && d < hd) a.out[(size_t)qi * a.ldo + (size_t)h * hd + d] = (uint16_t)cvt_bf16x2(acc[t] * inv, 0.0f);
    }
}

static int launch_any(const BlockAttnArgs &a) {
    const char *op = "attention_blocks";
    auto bytes = [](int hd) {
        return (size_t)kKeysPerTile * (hd + 2) * 2 + (size_t)kKeysPerTile * hd * 2 + (size_t)kQPerBlock * hd * 4;
    };
    if (a.head_dim > kMaxHeadDim) {
        set_error(IRIS_B200_EUNSUPPORTED, op, "head_dim above 512");
        return IRIS_B200_EUNSUPPORTED;
    }
    const int tiles = ((a.q_block < a.seq_q ? a.q_block : a.seq_q) + kQPerBlock - 1) / kQPerBlock;
    if ((long long)tiles * a.q_blocks > INT_MAX) {
        set_error(IRIS_B200_EUNSUPPORTED, op, "too many query tiles");
        return IRIS_B200_EUNSUPPORTED;
    }
    if (bytes(a.head_dim) > 48 * 1024 &&
        !cuda_ok(cudaFuncSetAttribute(k_attention_blocks_any, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(kMaxHeadDim)),
                 op))
        return IRIS_B200_ECUDA;
    k_attention_blocks_any<<<dim3((unsigned)(tiles * a.q_blocks), (unsigned)a.heads), kQPerBlock * 32, bytes(a.head_dim), g.stream>>>(
        a, tiles);
    return after_launch(op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}

}  // namespace iris_b200

using namespace iris_b200;

extern "C" int iris_b200_attention_blocks(uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k,
                                          int ldk, const uint16_t *v, int ldv, int seq_q, int seq_k, int heads, int kv_heads,
                                          int head_dim, float scale, const int *key_mask, const int *list, int list_len,
                                          int q_block, int k_block, int kernel) {
    const char *op = "attention_blocks";
    auto bad = [op](const char *why) {
        set_error(IRIS_B200_EINVAL, op, why);
        return (int)IRIS_B200_EINVAL;
    };
    if (seq_q < 0 || seq_k < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || list_len < 0 ||
        q_block <= 0 || k_block <= 0)
        return bad("bad argument");
    if ((long long)heads * head_dim > ldo || (long long)heads * head_dim > ldq || (long long)kv_heads * head_dim > ldk ||
        (long long)kv_heads * head_dim > ldv)
        return bad("a row stride is shorter than a row of heads");
    if (!(scale > 0.0f) || scale > 3.0e38f) return bad("scale must be positive and finite");
    if (kernel < IRIS_B200_KERNEL_AUTO || kernel > IRIS_B200_KERNEL_GENERIC) return bad("unknown kernel");
    if (heads > 65535) return bad("too many heads");
    if (list_len > 1 << 30) return bad("list_len above 2^30");
    if (seq_q > 0 && (!out || !q || (seq_k > 0 && (!k || !v)) || (list_len > 0 && !list))) return bad("bad argument");
    BlockAttnArgs a = {};
    a.out = out;
    a.ldo = ldo;
    a.q = q;
    a.ldq = ldq;
    a.k = k;
    a.ldk = ldk;
    a.v = v;
    a.ldv = ldv;
    a.seq_q = seq_q;
    a.seq_k = seq_k;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.key_mask = key_mask;
    a.list = list;
    a.list_len = list_len;
    a.q_block = q_block;
    a.k_block = k_block;
    a.q_blocks = (int)(((long long)seq_q + q_block - 1) / q_block);
    a.k_blocks = (int)(((long long)seq_k + k_block - 1) / k_block);
    const bool fast = attention_blocks_sm100_supported(a);
    if (kernel == IRIS_B200_KERNEL_TCGEN05 && !fast) {
        set_error(IRIS_B200_EUNSUPPORTED, op, "arguments outside the tcgen05 kernel's domain");
        return IRIS_B200_EUNSUPPORTED;
    }
    if (!require_device(op)) return IRIS_B200_ENODEV;
    if (seq_q == 0) return IRIS_B200_OK;
    if (kernel == IRIS_B200_KERNEL_AUTO && attention_blocks_row_supported(a)) return launch_attention_blocks_row(a);
    return fast && kernel != IRIS_B200_KERNEL_GENERIC ? launch_attention_blocks_sm100(a) : launch_any(a);
}
