/*
 * Which key blocks a query block attends to: block means of Q and K rows, and
 * the lists of the best-scoring key blocks.
 *
 * k_block_means reads every element once and is bound by HBM. A CTA owns one
 * block of rows and 256 columns, 32 lanes x 16 bytes; its eight warps take
 * every eighth row. A thread adds up to sixteen rows in fp32 and joins these
 * partial sums, and then the warps', in fp64, so that a mean is off by no more
 * than the rounding of a few sixteen-row sums.
 *
 * k_block_select scores in fp64: a product of two fp32 means is exact there,
 * and a list only depends on the order of summation where two scores agree to
 * 1e-16. Rows of a score tile are eight (query block, head) pairs of one key
 * head; the products run on the fp64 matrix instruction (m8n8k4), whose
 * operand fragments are read straight from the fp32 means: the summation
 * index may be permuted as long as both operands agree, so a lane takes four
 * consecutive dimensions with one 16-byte load and no shared memory is needed.
 * The scores become order-preserving 64-bit keys in shared memory; a warp then
 * finds the topk-th largest key of a row by bisection over its bits and writes
 * the chosen blocks in ascending order, equal keys from the lowest index.
 */
#include "common.cuh"

#include <limits.h>

#include "iris_dev.h"

namespace iris_b200 {
namespace block_select {

/* ---- block means ---- */

static constexpr int kMeanThreads = 256;
static constexpr int kMeanCols = 256;            /* columns of a CTA */
static constexpr int kMeanRun = 16;              /* rows of a thread summed in fp32 */

/* VEC: 16-byte loads (head_dim and strides multiples of 8, aligned base). */
template <bool VEC>
__global__ void __launch_bounds__(kMeanThreads)
k_block_means(float *__restrict__ means, int *__restrict__ counts, const uint16_t *__restrict__ x, int ldx, int seq,
              int width, int block, const int *__restrict__ row_mask) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double part[8][kMeanCols];
    __shared__ int part_n[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = blockIdx.y * kMeanCols + lane * 8;
    const long long r0 = (long long)blockIdx.x * block;
    const int rows = (int)(seq - r0 < block ? seq - r0 : block);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    double acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = 0.0;
    int n = 0;
    for (int rb = warp; rb < rows; rb += 8 * kMeanRun) {
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = 0.0f;
#pragma unroll
        for (int b = 0; b < kMeanRun; b += 8) {
            uint4 v[8];
            bool ok[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = rb + (b + i) * 8;
                ok[i] = r < rows && (!row_mask || __ldg(row_mask + r0 + r) != 0);
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (!ok[i]) continue;
                const uint16_t *src = x + (size_t)(r0 + r) * ldx + c0;
                if (VEC) {
                    if (c0 < width) v[i] = __ldg(reinterpret_cast<const uint4 *>(src));
                } else {
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (c0 + e < width) w[e >> 1] |= (uint32_t)src[e] << (16 * (e & 1));
                    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                n += ok[i];
                s[0] += bf_lo(v[i].x); s[1] += bf_hi(v[i].x);
                s[2] += bf_lo(v[i].y); s[3] += bf_hi(v[i].y);
                s[4] += bf_lo(v[i].z); s[5] += bf_hi(v[i].z);
                s[6] += bf_lo(v[i].w); s[7] += bf_hi(v[i].w);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] += (double)s[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) part[warp][lane * 8 + i] = acc[i];
    if (lane == 0) part_n[warp] = n;
    __syncthreads();
    const int c = blockIdx.y * kMeanCols + threadIdx.x;
    double sum = 0.0;
    int total = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        sum += part[w][threadIdx.x];
        total += part_n[w];
    }
    if (c < width) means[(size_t)blockIdx.x * width + c] = total ? (float)(sum / total) : 0.0f;
    if (counts && blockIdx.y == 0 && threadIdx.x == 0) counts[blockIdx.x] = total;
}

/* ---- lists ---- */

static constexpr int kSelThreads = 256;
static constexpr int kSelRows = 8;               /* (query block, head) rows of a CTA */
static constexpr int kMaxBlocks = 24576;         /* 64-bit keys of one row in shared memory */

struct Select {
    int *list;
    const float *qm, *km;
    const int *counts;
    int q_blocks, k_blocks, heads, kv_heads, head_dim;
    int group;                  /* query heads of a key head */
    int topk, keep_first, keep_last;
    int rows;                   /* rows of a CTA: kSelRows, or fewer where their keys would not fit */
};

__device__ __forceinline__ unsigned long long key_of(double s) {
    if (s != s) s = -__longlong_as_double(0x7FF0000000000000ll);        /* NaN ranks last */
    s += 0.0;                                                           /* -0 and +0 are equal */
    const unsigned long long b = (unsigned long long)__double_as_longlong(s);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

/* Row r of key head g: the query block and head. Rows run over the heads of
 * the group inside a query block, so the lists of a tile lie close together. */
__device__ __forceinline__ bool row_of(const Select &p, int g, long long r, int *qb, int *head) {
    if (r >= (long long)p.q_blocks * p.group) return false;
    *qb = (int)(r / p.group);
    *head = g * p.group + (int)(r - (long long)*qb * p.group);
    return true;
}

/* Scores of the rows r0 .. r0 + 7 of key head g against the blocks j0 .. j0 + 7
 * by one warp: two fp64 values per lane, row lane / 4, blocks j0 + 2 (lane & 3)
 * and the next. VEC: four consecutive dimensions per lane and step. */
template <bool VEC>
__device__ __forceinline__ void score_tile(const Select &p, const float *qrow, const float *krow, int lane, double d[2]) {
    d[0] = d[1] = 0.0;
    for (int k0 = 0; k0 < p.head_dim; k0 += 16) {
        const int e = k0 + (lane & 3) * 4;
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (VEC) {
            if (qrow) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(qrow + e));
                a[0] = v.x; a[1] = v.y; a[2] = v.z; a[3] = v.w;
            }
            if (krow) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(krow + e));
                b[0] = v.x; b[1] = v.y; b[2] = v.z; b[3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (qrow && e + i < p.head_dim) a[i] = qrow[e + i];
                if (krow && e + i < p.head_dim) b[i] = krow[e + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double av = (double)a[i], bv = (double)b[i];
            asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                         : "+d"(d[0]), "+d"(d[1]) : "d"(av), "d"(bv));
        }
    }
}

/* The list of one row by one warp: the keys of all blocks are in shared
 * memory (0: not eligible, all ones: always taken). */
__device__ __forceinline__ void choose(const Select &p, const unsigned long long *keys, int *list, int lane) {
    int eligible = 0;
    unsigned long long hi = 0ull, lo = ~0ull;
    for (int j = lane; j < p.k_blocks; j += 32) {
        const unsigned long long k = keys[j];
        eligible += k != 0ull;
        hi = k > hi ? k : hi;
        lo = k != 0ull && k < lo ? k : lo;
    }
    eligible = __reduce_add_sync(0xffffffffu, eligible);
    int want = p.topk < eligible ? p.topk : eligible;
    unsigned long long cut = 1ull;               /* keys above the cut are taken, equal ones from the lowest index */
    if (want < eligible) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long a = __shfl_xor_sync(0xffffffffu, hi, o), b = __shfl_xor_sync(0xffffffffu, lo, o);
            hi = a > hi ? a : hi;
            lo = b < lo ? b : lo;
        }
        /* The largest value that at least `want` keys reach: lo is reached by all, and the answer is not above hi. */
        while (lo < hi) {
            const unsigned long long mid = hi - ((hi - lo) >> 1);        /* lo < mid <= hi */
            int n = 0;
            for (int j = lane; j < p.k_blocks; j += 32) n += keys[j] >= mid;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= want)
                lo = mid;
            else
                hi = mid - 1ull;
            if (n == want) break;
        }
        cut = lo;
    }
    int above = 0;
    for (int j = lane; j < p.k_blocks; j += 32) above += keys[j] > cut;
    above = __reduce_add_sync(0xffffffffu, above);
    int equal_left = want - above;               /* of the keys equal to the cut */
    int done = 0;
    for (int j0 = 0; j0 < p.k_blocks && done < want; j0 += 32) {
        const unsigned long long k = j0 + lane < p.k_blocks ? keys[j0 + lane] : 0ull;
        const unsigned eq = __ballot_sync(0xffffffffu, k != 0ull && k == cut);
        const unsigned before = (1u << lane) - 1u;
        const bool take = k != 0ull && (k > cut || (k == cut && __popc(eq & before) < equal_left));
        const unsigned m = __ballot_sync(0xffffffffu, take);
        if (take) list[done + __popc(m & before)] = j0 + lane;
        done += __popc(m);
        equal_left -= __popc(eq) < equal_left ? __popc(eq) : equal_left;
    }
    for (int i = want + lane; i < p.topk; i += 32) list[i] = -1;
}

template <bool VEC>
__global__ void __launch_bounds__(kSelThreads)
k_block_select(const __grid_constant__ Select p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ unsigned long long keys[];         /* [rows][k_blocks] */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = blockIdx.y;
    const long long r0 = (long long)blockIdx.x * p.rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int qb, head;
    const int mine = lane >> 2;                          /* row of the score tile this lane feeds and receives */
    const bool live = mine < p.rows && row_of(p, g, r0 + mine, &qb, &head);
    const float *qrow = live ? p.qm + ((size_t)qb * p.heads + head) * p.head_dim : nullptr;
    for (int j0 = warp * 8; j0 < p.k_blocks; j0 += (kSelThreads / 32) * 8) {
        const int jb = j0 + mine;
        const float *krow = jb < p.k_blocks ? p.km + ((size_t)jb * p.kv_heads + g) * p.head_dim : nullptr;
        double d[2];
        score_tile<VEC>(p, qrow, krow, lane, d);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int j = j0 + (lane & 3) * 2 + i;
            if (mine < p.rows && j < p.k_blocks) {
                const bool ok = !p.counts || __ldg(p.counts + j) > 0;
                const bool kept = j < p.keep_first || j >= p.k_blocks - p.keep_last;
                keys[(size_t)mine * p.k_blocks + j] = !ok ? 0ull : (kept ? ~0ull : key_of(d[i]));
            }
        }
    }
    __syncthreads();
    for (int r = warp; r < p.rows; r += kSelThreads / 32)
        if (row_of(p, g, r0 + r, &qb, &head))
            choose(p, keys + (size_t)r * p.k_blocks, p.list + ((size_t)head * p.q_blocks + qb) * p.topk, lane);
}

static int g_select_ready = 0;

static int bad(const char *op, const char *why) {
    set_error(IRIS_B200_EINVAL, op, why);
    return IRIS_B200_EINVAL;
}
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

/* Launch with programmatic stream serialisation: both kernels wait for the grid ahead before they touch memory. */
static void configure(cudaLaunchConfig_t *cfg, cudaLaunchAttribute *attr, dim3 grid, int threads, size_t smem) {
    cfg->gridDim = grid;
    cfg->blockDim = dim3(threads);
    cfg->dynamicSmemBytes = smem;
    cfg->stream = g.stream;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

}  // namespace block_select

void block_select_release(void) { block_select::g_select_ready = 0; }

}  // namespace iris_b200

using namespace iris_b200;
using namespace iris_b200::block_select;

extern "C" int iris_b200_block_means(float *means, int *counts, const uint16_t *x, int ldx, int seq, int heads, int head_dim,
                                     int block, const int *row_mask) {
    const char *op = "block_means";
    if (seq < 0 || heads <= 0 || head_dim <= 0 || block <= 0 || (long long)heads * head_dim > ldx) return bad(op, "bad argument");
    if (seq > 0 && (!means || !x)) return bad(op, "bad argument");
    const int width = heads * head_dim;
    const int tiles = (width + kMeanCols - 1) / kMeanCols;
    if (tiles > 65535) return bad(op, "too many columns");
    if (!require_device(op)) return IRIS_B200_ENODEV;
    if (seq == 0) return IRIS_B200_OK;
    const bool vec = width % 8 == 0 && ldx % 8 == 0 && aligned16(x);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    configure(&cfg, &attr, dim3((unsigned)(((long long)seq + block - 1) / block), (unsigned)tiles), kMeanThreads, 0);
    const cudaError_t err = cudaLaunchKernelEx(&cfg, vec ? k_block_means<true> : k_block_means<false>, means, counts, x, ldx, seq,
                                               width, block, row_mask);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}

extern "C" int iris_b200_block_select(int *list, const float *q_means, const float *k_means, const int *k_counts, int q_blocks,
                                      int k_blocks, int heads, int kv_heads, int head_dim, int topk, int keep_first,
                                      int keep_last) {
    const char *op = "block_select";
    if (q_blocks < 0 || k_blocks < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 || topk <= 0 ||
        keep_first < 0 || keep_last < 0)
        return bad(op, "bad argument");
    if ((long long)keep_first + keep_last > topk) return bad(op, "more blocks to keep than the list holds");
    if (kv_heads > 65535) return bad(op, "too many key heads");
    if (k_blocks > kMaxBlocks) {
        set_error(IRIS_B200_EUNSUPPORTED, op, "more than 24576 key blocks");
        return IRIS_B200_EUNSUPPORTED;
    }
    if (q_blocks > 0 && (!list || !q_means || (k_blocks > 0 && !k_means))) return bad(op, "bad argument");
    if (!require_device(op)) return IRIS_B200_ENODEV;
    if (q_blocks == 0) return IRIS_B200_OK;
    Select p = {};
    p.list = list;
    p.qm = q_means;
    p.km = k_means;
    p.counts = k_counts;
    p.q_blocks = q_blocks;
    p.k_blocks = k_blocks;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.head_dim = head_dim;
    p.group = heads / kv_heads;
    p.topk = topk;
    p.keep_first = keep_first < k_blocks ? keep_first : k_blocks;
    p.keep_last = keep_last < k_blocks ? keep_last : k_blocks;
    p.rows = kSelRows;
    while (p.rows > 1 && p.rows * k_blocks > kMaxBlocks) p.rows--;
    const bool vec = head_dim % 16 == 0 && aligned16(q_means) && aligned16(k_means);
    const size_t smem = (size_t)p.rows * k_blocks * 8;
    if (!g_select_ready) {
        if (!cuda_ok(cudaFuncSetAttribute(k_block_select<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBlocks * 8), op) ||
            !cuda_ok(cudaFuncSetAttribute(k_block_select<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBlocks * 8), op))
            return IRIS_B200_ECUDA;
        g_select_ready = 1;
    }
    const long long rows = (long long)q_blocks * p.group, tiles = (rows + p.rows - 1) / p.rows;
    if (tiles > INT_MAX) return bad(op, "too many query blocks");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    configure(&cfg, &attr, dim3((unsigned)tiles, (unsigned)kv_heads), kSelThreads, smem);
    const cudaError_t err = cudaLaunchKernelEx(&cfg, vec ? k_block_select<true> : k_block_select<false>, p);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}
