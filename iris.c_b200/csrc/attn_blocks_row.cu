/*
 * Attention over lists of key blocks where every query row has a list of its
 * own: single tokens at the end of a long cache, or a list per token.
 *
 * A tensor-core tile would hold one row of 128, and its chain of copy, scores,
 * softmax and product leaves the memory idle between tiles. Here the keys are
 * read straight into registers and multiplied on the CUDA cores, so that many
 * warps keep loads in flight. LANES = head_dim / 8 lanes hold one K or V row,
 * 16 bytes each; a warp takes a chunk of KEYS = 8 * 32 / LANES keys at a time
 * with all its K and V rows (8 KB) under way at once. The partial products of
 * eight keys are summed over their lanes by an exchange that halves the number
 * of values in every step, after which a lane owns one key's score.
 *
 * Maximum, sum and accumulators are fp32 and private to a warp; probabilities
 * are not rounded. The chunks of a list go round the warps of a cluster of up
 * to sixteen CTAs, whose results meet in shared memory: first in each CTA,
 * then in the first one.
 *
 * Bound by HBM where the lists of a call do not fit in L2: one row of 32 heads
 * over 64 blocks of 64 keys each reads 67 MB (61 MB of different rows, where four
 * heads share a key head and their lists overlap) in 14.8 us back to back (4.5
 * TB/s); with head_dim 256, 134 MB, 24.4 us, so that 67 MB more cost 9.6 us (7.0
 * TB/s) and 5 us are launch, list, first loads and joining. The tensor-core
 * kernel takes 19.1 us for the former, and for 256 rows of 32 heads over 32
 * blocks, out of L2, 893 us against 712. Half as many loads per warp and twice
 * the warps: 20.8 us; the next chunk's loads started under the products of
 * this one, which spills: 15.0 us and 856 us.
 */
#include "common.cuh"

#include <limits.h>
#include <math.h>

#include "kernels.h"
#include "tc_ptx.cuh"

namespace iris_b200 {
namespace attn_row {

using namespace sm100;

static constexpr int kThreads = 256;
static constexpr int kWarps = kThreads / 32;
static constexpr int kCtasPerSM = 2;
static constexpr int kMaxParts = 16;              /* CTAs of a cluster, where the device takes as many */
static constexpr int kLoads = 8;                 /* K rows of a lane in flight, and as many V rows */

struct Params {
    BlockAttnArgs a;
    int chunks_per_entry, chunks;                /* of a list entry, of a list */
    int parts;                                   /* CTAs of a cluster */
    float scale_log2;
};

/* Sums over the lanes of a row of eight values each: lane l gets the sum of value index_of(l). */
template <int LANES>
__device__ __forceinline__ float sum_rows(float s[kLoads], int lane) {
    int o = LANES / 2;
#pragma unroll
    for (int n = kLoads / 2; n >= 1; n >>= 1, o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float give = upper ? s[i] : s[i + n], keep = upper ? s[i + n] : s[i];
            s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (; o >= 1; o >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    return s[0];
}

template <int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSM)
k_attention_blocks_row(const __grid_constant__ Params p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int LANES = HD / 8, GROUPS = 32 / LANES, KEYS = kLoads * GROUPS;
    constexpr int SPREAD = LANES / kLoads;       /* neighbouring lanes that own the same key */
    __shared__ float part[kWarps][HD];
    __shared__ float2 part_ml[kWarps];
    __shared__ float cta[HD];
    __shared__ float2 cta_ml;
    const BlockAttnArgs &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (LANES - 1), grp = lane / LANES;
    const int rank = p.parts > 1 ? (int)cluster_cta_rank() : 0;
    const int row = (int)(blockIdx.x / (unsigned)p.parts), head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads);
    const uint16_t *kbase = a.k + (size_t)kv_head * HD + l * 8, *vbase = a.v + (size_t)kv_head * HD + l * 8;
    const int *list = a.list + ((size_t)head * a.q_blocks + row) * a.list_len;
    const int mine = (l / SPREAD) * GROUPS + grp;              /* the key of a chunk that this lane owns */
    /* Started under the kernel ahead: what it wrote is read after its end, and by plain loads. */
    asm volatile("griddepcontrol.wait;" ::: "memory");

    float q[8];
    {
        const uint4 v = *reinterpret_cast<const uint4 *>(a.q + (size_t)row * a.ldq + (size_t)head * HD + l * 8);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[2 * i] = bf_lo(w[i]) * p.scale_log2;
            q[2 * i + 1] = bf_hi(w[i]) * p.scale_log2;
        }
    }
    float m = -INFINITY, sum = 0.0f, acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = 0.0f;

    /* A warp's chunks are gw, gw + stride, ...; a lane looks up one of the next 32. */
    const int stride = p.parts * kWarps;
    for (int base = rank * kWarps + warp; base < p.chunks; base += 32 * stride) {
        const int c = base + lane * stride;
        int first = 0, rows = 0;
        if (c < p.chunks) {
            const int e = c / p.chunks_per_entry, k0 = (c - e * p.chunks_per_entry) * KEYS;
            const int b = list[e];
            if (b >= 0 && b < a.k_blocks) {
                const long long f = (long long)b * a.k_block + k0;
                const long long n = a.seq_k - f < a.k_block - k0 ? a.seq_k - f : a.k_block - k0;
                if (n > 0) {
                    first = (int)f;
                    rows = n < KEYS ? (int)n : KEYS;
                }
            }
        }
        unsigned todo = __ballot_sync(0xffffffffu, rows > 0);
        while (todo) {
            const int src = __ffs(todo) - 1;
            todo &= todo - 1;
            const int key0 = __shfl_sync(0xffffffffu, first, src), n = __shfl_sync(0xffffffffu, rows, src);
            uint4 kr[kLoads], vr[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int key = i * GROUPS + grp;
                kr[i] = make_uint4(0u, 0u, 0u, 0u);
                if (key < n) kr[i] = *reinterpret_cast<const uint4 *>(kbase + (size_t)(key0 + key) * a.ldk);
            }
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int key = i * GROUPS + grp;
                vr[i] = make_uint4(0u, 0u, 0u, 0u);
                if (key < n) vr[i] = *reinterpret_cast<const uint4 *>(vbase + (size_t)(key0 + key) * a.ldv);
            }
            unsigned valid = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
            if (a.key_mask) valid = __ballot_sync(0xffffffffu, lane < n && a.key_mask[key0 + (lane < n ? lane : 0)] != 0);

            float s[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const uint32_t w[4] = {kr[i].x, kr[i].y, kr[i].z, kr[i].w};
                float x = 0.0f, y = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x = fmaf(q[2 * j], bf_lo(w[j]), x);
                    y = fmaf(q[2 * j + 1], bf_hi(w[j]), y);
                }
                s[i] = x + y;
            }
            float score = sum_rows<LANES>(s, lane);
            if (!((valid >> mine) & 1u)) score = -INFINITY;
            float mx = score;
#pragma unroll
            for (int o = 16; o >= SPREAD; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mnew = fmaxf(m, mx), ref = mnew == -INFINITY ? 0.0f : mnew;
            const float alpha = ex2(m - ref), pr = ex2(score - ref);
            m = mnew;
            sum = fmaf(sum, alpha, pr);
#pragma unroll
            for (int i = 0; i < 8; i++) acc[i] *= alpha;
            if (a.key_mask) {
                /* A zero probability does not cancel a NaN. */
#pragma unroll
                for (int i = 0; i < kLoads; i++)
                    if (!((valid >> (i * GROUPS + grp)) & 1u)) vr[i] = make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const float pi = __shfl_sync(0xffffffffu, pr, grp * LANES + i * SPREAD);
                const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    acc[2 * j] = fmaf(pi, bf_lo(w[j]), acc[2 * j]);
                    acc[2 * j + 1] = fmaf(pi, bf_hi(w[j]), acc[2 * j + 1]);
                }
            }
        }
    }

    /* The lanes of a warp, its groups, the warps, the CTAs. */
#pragma unroll
    for (int o = 16; o >= SPREAD; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    }
    if (grp == 0) {
        float4 *dst = reinterpret_cast<float4 *>(&part[warp][l * 8]);
        dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
    if (lane == 0) part_ml[warp] = make_float2(m, sum);
    __syncthreads();
    const int d = threadIdx.x;
    uint16_t *out = a.out + (size_t)row * a.ldo + (size_t)head * HD;
    float mc = -INFINITY, lc = 0.0f, oc = 0.0f;
    if (d < HD) {
#pragma unroll
        for (int w = 0; w < kWarps; w++) mc = fmaxf(mc, part_ml[w].x);
        const float ref = mc == -INFINITY ? 0.0f : mc;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = ex2(part_ml[w].x - ref);
            lc = fmaf(part_ml[w].y, f, lc);
            oc = fmaf(part[w][d], f, oc);
        }
    }
    if (p.parts == 1) {
        if (d < HD) out[d] = (uint16_t)cvt_bf16x2(lc != 0.0f ? oc / lc : 0.0f, 0.0f);
        return;
    }
    if (d < HD) cta[d] = oc;
    if (d == 0) cta_ml = make_float2(mc, lc);
    cluster_sync_all();
    if (rank == 0 && d < HD) {
        float2 ml[kMaxParts];
        float o[kMaxParts];
        float mt = -INFINITY, lt = 0.0f, ot = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxParts; r++) {
            ml[r] = make_float2(-INFINITY, 0.0f);
            o[r] = 0.0f;
            if (r < p.parts) {
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                             : "=f"(ml[r].x), "=f"(ml[r].y) : "r"(map_to_cta(smem_u32(&cta_ml), r)) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[r]) : "r"(map_to_cta(smem_u32(&cta[d]), r)) : "memory");
            }
        }
#pragma unroll
        for (int r = 0; r < kMaxParts; r++) mt = fmaxf(mt, ml[r].x);
        const float ref = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
        for (int r = 0; r < kMaxParts; r++) {
            const float f = ex2(ml[r].x - ref);
            lt = fmaf(ml[r].y, f, lt);
            ot = fmaf(o[r], f, ot);
        }
        out[d] = (uint16_t)cvt_bf16x2(lt != 0.0f ? ot / lt : 0.0f, 0.0f);
    }
    __syncwarp();
    cluster_sync_all();                          /* nobody leaves while its sums are being read */
}

static int g_max_parts = 0;                      /* 0: not asked yet */

/* Sixteen CTAs are more than every device promises a cluster: 1 head over 128
 * blocks of 64 keys takes 7.9 us so, 12.0 us with eight; 8 heads over 64 blocks
 * 7.7 and 9.3 us. */
static int max_parts() {
    if (g_max_parts) return g_max_parts;
    auto allow = [](auto kernel) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    };
    int parts = 8;
    if (allow(k_attention_blocks_row<64>) && allow(k_attention_blocks_row<128>) && allow(k_attention_blocks_row<256>)) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(kMaxParts);
        cfg.blockDim = dim3(kThreads);
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kMaxParts;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int fit = 0;
        if (cudaOccupancyMaxActiveClusters(&fit, k_attention_blocks_row<256>, &cfg) == cudaSuccess && fit > 0) parts = kMaxParts;
    }
    if (parts < kMaxParts) (void)cudaGetLastError();     /* a refusal here is an answer, not an error */
    return g_max_parts = parts;
}

/* Keys of a chunk. */
static int chunk_keys(int head_dim) { return kLoads * 32 / (head_dim / 8); }

static long long chunks_of(const BlockAttnArgs &a) {
    const int keys = chunk_keys(a.head_dim), block = a.k_block < a.seq_k ? a.k_block : a.seq_k;
    return (long long)a.list_len * ((block + keys - 1) / keys);
}

}  // namespace attn_row

void attention_blocks_row_release(void) { attn_row::g_max_parts = 0; }

bool attention_blocks_row_supported(const BlockAttnArgs &a) {
    const uintptr_t bits = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
    return (a.q_block == 1 || a.seq_q == 1) && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && a.ldq % 8 == 0 &&
           a.ldk % 8 == 0 && a.ldv % 8 == 0 && (bits & 15) == 0 && a.seq_k > 0 && a.seq_q <= INT_MAX / attn_row::kMaxParts &&
           attn_row::chunks_of(a) <= INT_MAX - 32 * attn_row::kMaxParts * attn_row::kWarps;
}

int launch_attention_blocks_row(const BlockAttnArgs &a) {
    using namespace attn_row;
    Params p = {};
    p.a = a;
    p.chunks = (int)chunks_of(a);
    p.chunks_per_entry = a.list_len > 0 ? p.chunks / a.list_len : 1;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    /* The list of a row is cut over the CTAs of a cluster while the device has
     * room for more and every warp keeps a chunk. */
    const long long items = (long long)a.heads * a.seq_q;
    p.parts = 1;
    while (p.parts < max_parts() && items * p.parts * 2 <= (long long)kCtasPerSM * g.sm_count && p.chunks >= p.parts * 2 * kWarps) p.parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.seq_q * p.parts), (unsigned)a.heads);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = g.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.parts;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.parts > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, a.head_dim == 64    ? k_attention_blocks_row<64>
                                                     : a.head_dim == 128 ? k_attention_blocks_row<128>
                                                                         : k_attention_blocks_row<256>, p);
    g.launches++;
    return cuda_ok(err, "attention_blocks") ? IRIS_B200_OK : IRIS_B200_ECUDA;
}

}  // namespace iris_b200
