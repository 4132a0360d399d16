/*
 * Which key blocks a query block attends to: block means of Q and K rows, and
 * the lists of the best-scoring key blocks.
 *
 * k_block_means reads every element once and is bound by HBM. A CTA owns one
 * block of rows and 256 columns, 32 lanes x 16 bytes; its eight warps take
 * every eighth row. A thread adds up to eight rows in fp32, an eighth of each
 * (exact in fp32 for every bf16 value, and eight of the largest do not overflow),
 * and joins these partial sums, and then the warps', in fp64, so that a mean is
 * off by no more than the rounding of eight-row sums. 16 889 rows x 32 heads in blocks
 * of 128 (141 MB) take 23.8 us, 5.9 TB/s; 4608 x 30 in blocks of 64 (37 MB)
 * 8.9 us, less than two waves of CTAs.
 *
 * k_block_select scores in fp64: a product of two fp32 means is exact there,
 * and a list only depends on the order of summation where two scores agree to
 * 1e-16. Up to sixteen (query block, head) rows of one key head share a score
 * tile on the fp64 matrix instruction (m8n8k4). Its key operand is read
 * straight from the fp32 means: the summation index may be permuted as long as
 * both operands agree, so a lane takes four consecutive dimensions with one
 * 16-byte load and all loads of a tile are in flight together. The scores
 * become order-preserving 64-bit keys in shared memory. Where there are few
 * rows, the blocks are cut over the CTAs of a cluster, which send the keys to
 * the CTA that chooses for the row. One to eight warps then find the topk-th
 * largest key of a row, by a histogram and within its bin by rank, and write
 * the chosen blocks in ascending order, equal keys from the lowest index.
 * 132 query blocks x 32 heads over 264 blocks take 26.2 us: products about 14
 * (8 at the rate of the fp64 matrix pipe), the choice 3.3 a row, two rows a
 * warp. One query block of 32 heads on 8 key heads over 2048 blocks 11.9 us:
 * latency of the cluster's barriers, the loads and the choice. tf32 products
 * with an fp64 check of the cut were no faster.
 *
 * Both kernels start under the kernel ahead of them and wait for its end. What
 * they read may be written until then, so it is never read through the
 * non-coherent path, which takes memory as constant for the whole kernel: no
 * __ldg and no __restrict__ here.
 */
#include "common.cuh"

#include <limits.h>

#include "iris_dev.h"
#include "tc_ptx.cuh"

namespace iris_b200 {
namespace block_select {

/* ---- block means ---- */

static constexpr int kMeanThreads = 256;
static constexpr int kMeanCols = 256;            /* columns of a CTA */
static constexpr int kMeanRun = 8;               /* rows of a thread in flight, and summed in fp32 */

/* VEC: 16-byte loads (head_dim and strides multiples of 8, aligned base). */
template <bool VEC>
__global__ void __launch_bounds__(kMeanThreads, 4)
k_block_means(float *means, int *counts, const uint16_t *x, int ldx, int seq, int width, int block, const int *row_mask) {
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
    /* (Unsigned: rb may pass the last row by more than a 31-bit count has room for.) */
    for (unsigned rb = warp; rb < (unsigned)rows; rb += 8 * kMeanRun) {
        /* Which of the run's rows count (bit i: row rb + 8 i), then all their loads at once. */
        const unsigned mine = rb + 8 * lane;
        const bool counts_mine = lane < kMeanRun && mine < (unsigned)rows && (!row_mask || row_mask[r0 + mine] != 0);
        const unsigned ok = __ballot_sync(0xffffffffu, counts_mine);
        n += __popc(ok);
        uint4 v[kMeanRun];
#pragma unroll
        for (int i = 0; i < kMeanRun; i++) {
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (!((ok >> i) & 1u)) continue;
            const uint16_t *src = x + (size_t)(r0 + rb + 8 * i) * ldx + c0;
            if (VEC) {
                if (c0 < width) v[i] = *reinterpret_cast<const uint4 *>(src);
            } else {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c0 + e < width) w[e >> 1] |= (uint32_t)src[e] << (16 * (e & 1));
                v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < kMeanRun; i++) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[2 * e] = fmaf(bf_lo(w[e]), 1.0f / kMeanRun, s[2 * e]);
                s[2 * e + 1] = fmaf(bf_hi(w[e]), 1.0f / kMeanRun, s[2 * e + 1]);
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
    if (c < width) means[(size_t)blockIdx.x * width + c] = total ? (float)(sum * kMeanRun / total) : 0.0f;
    if (counts && blockIdx.y == 0 && threadIdx.x == 0) counts[blockIdx.x] = total;
}

/* ---- lists ---- */

static constexpr int kSelThreads = 256;
static constexpr int kSelWarps = kSelThreads / 32;
static constexpr int kSelRows = 16;              /* (query block, head) rows of a cluster: two score tiles of eight */
static constexpr int kMaxCtas = 16;              /* CTAs of a cluster, each with a slice of the blocks */
static constexpr int kWideSmem = 96 * 1024;      /* of a CTA in a cluster of more than eight: two CTAs fit an SM */
static constexpr int kMaxBlocks = 23552;         /* 64-bit keys of one row in shared memory */
static constexpr int kMaxHeadDim = 512;
static constexpr int kSelSmem = kMaxBlocks * 8 + kMaxHeadDim * 64;      /* one row's keys, one tile of rows */

struct Select {
    int *list;
    const float *qm, *km;
    const int *counts;
    int q_blocks, k_blocks, heads, kv_heads, head_dim;
    int group;                  /* query heads of a key head */
    int topk, keep_first, keep_last;
    int rows;                   /* rows of a cluster */
    int ctas, slice;            /* CTAs of a cluster, blocks of each (a multiple of 8) */
    int own_rows;               /* rows whose keys a CTA holds: ceil(rows / ctas) */
    int team;                   /* warps that choose for one row */
    int steps;                  /* products of four dimensions: head_dim rounded up to 16, / 4 */
};

__device__ __forceinline__ unsigned long long key_of(double s) {
    if (s != s) s = -__longlong_as_double(0x7FF0000000000000ll);        /* NaN ranks last */
    s += 0.0;                                                           /* -0 and +0 are equal */
    const unsigned long long b = (unsigned long long)__double_as_longlong(s);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

/* Row r of key head g: the query block and head. Rows run over the heads of
 * the group inside a query block. */
__device__ __forceinline__ bool row_of(const Select &p, int g, long long r, int *qb, int *head) {
    if (r >= (long long)p.q_blocks * p.group) return false;
    *qb = (int)(r / p.group);
    *head = g * p.group + (int)(r - (long long)*qb * p.group);
    return true;
}

__device__ __forceinline__ void mma_f64(double d[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

/* What a lane needs of a block for a score tile: four dimensions of every
 * sixteen. HD 0: any head_dim, read where it is used. */
template <int HD>
struct Block {
    float4 v[HD / 16 + 1];
    const float *row;
    __device__ __forceinline__ void load(const float *krow, int lane) {
        row = krow;
#pragma unroll
        for (int g = 0; g < HD / 16; g++)
            v[g] = krow ? *reinterpret_cast<const float4 *>(krow + 16 * g + (lane & 3) * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
};

/* Scores of the cluster's rows against eight blocks by one warp: d[m] holds row
 * 8 m + lane / 4 and the blocks 2 (lane & 3), + 1. Product s of a 16-dimension
 * group takes the dimensions 16 g + 4 (lane & 3) + s. qf: the rows as fp64 operand
 * fragments in shared memory. */
template <int HD>
__device__ __forceinline__ void score_tile(const Select &p, const double *qf, const Block<HD> &k, int lane, int tiles, double d[2][2]) {
    d[0][0] = d[0][1] = d[1][0] = d[1][1] = 0.0;
    if (HD > 0) {
        /* (Several sums per tile, so that a product does not wait for the one before.) */
        double more[3][2] = {{0.0, 0.0}, {0.0, 0.0}, {0.0, 0.0}};
        if (tiles > 1) {
#pragma unroll
            for (int g = 0; g < HD / 16; g++) {
                const float b[4] = {k.v[g].x, k.v[g].y, k.v[g].z, k.v[g].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const double bv = (double)b[i];
                    mma_f64(i & 1 ? more[0] : d[0], qf[(4 * g + i) * 32 + lane], bv);
                    mma_f64(i & 1 ? more[1] : d[1], qf[(p.steps + 4 * g + i) * 32 + lane], bv);
                }
            }
            d[1][0] += more[1][0];
            d[1][1] += more[1][1];
        } else {
#pragma unroll
            for (int g = 0; g < HD / 16; g++) {
                const float b[4] = {k.v[g].x, k.v[g].y, k.v[g].z, k.v[g].w};
#pragma unroll
                for (int i = 0; i < 4; i++) mma_f64(i ? more[i - 1] : d[0], qf[(4 * g + i) * 32 + lane], (double)b[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) d[0][i] += more[1][i] + more[2][i];
        }
        d[0][0] += more[0][0];
        d[0][1] += more[0][1];
    } else {
        for (int s = 0; s < p.steps; s++) {
            const int e = (s >> 2) * 16 + (lane & 3) * 4 + (s & 3);
            const double bv = k.row && e < p.head_dim ? (double)k.row[e] : 0.0;
            mma_f64(d[0], qf[s * 32 + lane], bv);
            if (tiles > 1) mma_f64(d[1], qf[(p.steps + s) * 32 + lane], bv);
        }
    }
}

/* A team of p.team warps works on one row; `me` is the warp's place in it. */
struct Team {
    int me, warps, barrier;
    unsigned *counts;           /* [2][kSelWarps][2] shared words of this team */
    unsigned turn;
    __device__ __forceinline__ void sync() const {
        if (warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
    }
    /* The team's sums of two words, and what the warps before this one add to them. */
    __device__ __forceinline__ void sum(unsigned &a, unsigned &b, unsigned &a_before, unsigned &b_before) {
        a = __reduce_add_sync(0xffffffffu, a);
        b = __reduce_add_sync(0xffffffffu, b);
        a_before = b_before = 0u;
        if (warps == 1) return;
        unsigned *c = counts + (turn++ & 1u) * (2 * kSelWarps);
        if ((threadIdx.x & 31) == 0) {
            c[2 * me] = a;
            c[2 * me + 1] = b;
        }
        sync();
        a = b = 0u;
        for (int w = 0; w < warps; w++) {
            if (w == me) {
                a_before = a;
                b_before = b;
            }
            a += c[2 * w];
            b += c[2 * w + 1];
        }
    }
    /* The team's maxima of two words. */
    __device__ __forceinline__ void most(unsigned &a, unsigned &b) {
        a = __reduce_max_sync(0xffffffffu, a);
        b = __reduce_max_sync(0xffffffffu, b);
        if (warps == 1) return;
        unsigned *c = counts + (turn++ & 1u) * (2 * kSelWarps);
        if ((threadIdx.x & 31) == 0) {
            c[2 * me] = a;
            c[2 * me + 1] = b;
        }
        sync();
        for (int w = 0; w < warps; w++) {
            a = c[2 * w] > a ? c[2 * w] : a;
            b = c[2 * w + 1] > b ? c[2 * w + 1] : b;
        }
    }
};

static constexpr int kBins = 256;
/* Bin of a score. Monotone: each operation rounds monotonically; per = kBins / range may round up, hence the limit. */
__device__ __forceinline__ int bin_of(float f, float low, float per) {
    const int b = (int)((f - low) * per);
    return b < kBins - 1 ? b : kBins - 1;
}
/* Scratch of a team in shared memory. */
struct TeamScratch {
    alignas(16) unsigned hist[kBins];
    unsigned counts[4 * kSelWarps];
    unsigned found;
    int candidates[32];
};
static constexpr uint32_t kOut = 0u, kTaken = ~0u;       /* upper words of keys that are no scores */

/* The score of a key from its upper word, to 20 bits, as fp32 (clamped to its
 * range): never out of order. */
__device__ __forceinline__ float score_of(uint32_t high) {
    const uint32_t flip = ~(uint32_t)((int)high >> 31);             /* negative scores are stored inverted */
    uint32_t t = (high ^ flip) & 0x7FFFFFFFu;                       /* exponent and upper mantissa of the fp64 magnitude */
    t = t < 0x38000000u ? 0x38000000u : (t > 0x47EFFFFFu ? 0x47EFFFFFu : t);
    return __uint_as_float((t - 0x38000000u) << 3 | (flip & 0x80000000u));
}
__device__ __forceinline__ uint32_t high_of(const unsigned long long *key) { return reinterpret_cast<const uint32_t *>(key)[1]; }

/* The list of one row: its keys (0: not eligible, all ones: always taken) are
 * in shared memory, a run of them for every warp of the team. A histogram of
 * the scores over 256 equal bins between the lowest and the highest narrows the
 * place of the topk-th down to one bin, on the upper words of the keys alone.
 * Where only a part of that bin is wanted its keys are ranked in full: up to 32
 * by one warp, more by a search over their bits. The chosen keys of the bin are
 * turned into all ones, and everything above the bin is taken.
 * WORDS > 0: a lane holds that many upper words in registers, which covers the
 * run, and every pass over them is straight-line code. It is compiled for the
 * multiples of four up to sixteen, as places that hold no word cost as much as
 * those that do: 132 query blocks x 32 heads over 128 / 256 / 384 / 512 blocks
 * take 14.9 / 23.5 / 32.2 / 40.8 us, with sixteen words alone 18.0 / 25.5 / 33.1 /
 * 40.5, with the words read from shared memory in loops (WORDS 0) 16.1 / 26.3 /
 * 36.3 / 46.2. (Even counts: half a microsecond less where they round up by less,
 * for twice the code.) Longer runs go through the loops: 544 blocks 49.8 us. */
template <int WORDS>
__device__ __forceinline__ void choose(const Select &p, Team t, unsigned long long *keys, TeamScratch &sc, int *list) {
    const int lane = threadIdx.x & 31;
    const int run = ((p.k_blocks + t.warps - 1) / t.warps + 31) & ~31;
    const int j0 = t.me * run < p.k_blocks ? t.me * run : p.k_blocks;
    const int j1 = j0 + run < p.k_blocks ? j0 + run : p.k_blocks;
    const unsigned before = (1u << lane) - 1u;
    uint32_t words[WORDS > 0 ? WORDS : 1];
    if (WORDS > 0) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) words[i] = j0 + 32 * i + lane < j1 ? high_of(keys + j0 + 32 * i + lane) : kOut;
    }
    /* fn(i, block, word) for this lane's blocks, kOut behind the last. */
    auto each = [&](auto fn) {
        if (WORDS > 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i++) fn(i, j0 + 32 * i + lane, words[i]);
        } else {
            for (int j = j0 + lane; j < j1; j += 32) fn(0, j, high_of(keys + j));
        }
    };
    unsigned eligible = 0, kept = 0, x, y, top = 0, bottom = 0;
    each([&](int, int, uint32_t w) {
        eligible += w != kOut;
        kept += w == kTaken;
        const bool score = w != kOut && w != kTaken;
        top = score && w > top ? w : top;
        bottom = score && ~w > bottom ? ~w : bottom;
    });
    for (int i = t.me * 32 + lane; i < kBins / 4; i += t.warps * 32) reinterpret_cast<uint4 *>(sc.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (t.me == 0 && lane == 0) sc.found = 0u;
    __syncwarp();
    t.sum(eligible, kept, x, y);
    const unsigned want = (unsigned)p.topk < eligible ? (unsigned)p.topk : eligible;
    uint32_t bar = kOut;                         /* upper words above it are taken */
    if (want < eligible) {
        bar = kTaken - 1u;
        if (want > kept) {
            t.most(top, bottom);
            const unsigned left = want - kept;           /* places for scores */
            const float low = score_of(~bottom), range = score_of(top) - low;
            /* (Without a span, or an infinite one, everything is in bin 0.) */
            const float per = range > 0.0f && range < 1e30f ? (float)kBins / range : 0.0f;
            int bins[WORDS > 0 ? WORDS : 1];             /* -1: no score */
            auto bin_at = [&](uint32_t w) { return w == kOut || w == kTaken ? -1 : per > 0.0f ? bin_of(score_of(w), low, per) : 0; };
            each([&](int i, int, uint32_t w) {
                const int b = bin_at(w);
                if (WORDS > 0) bins[i] = b;
                if (b >= 0) atomicAdd(sc.hist + b, 1u);
            });
            __syncwarp();
            t.sync();
            /* Scores in the bins above mine, eight bins a lane from the top; one lane holds the bin of the last place. */
            unsigned n[8], mine = 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint4 v = *reinterpret_cast<const uint4 *>(sc.hist + kBins - 8 * lane - 4 * (i + 1));
                n[4 * i] = v.w;
                n[4 * i + 1] = v.z;
                n[4 * i + 2] = v.y;
                n[4 * i + 3] = v.x;
                mine += v.x + v.y + v.z + v.w;
            }
            unsigned above = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += v;
            }
            above -= mine;
            unsigned found = 0;                          /* bin + 1 in bits 0 to 8, places left in it above */
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (above < left && above + n[i] >= left) found = (unsigned)(kBins - (lane * 8 + i)) | (left - above) << 9 | (n[i] == left - above ? 1u << 31 : 0u);
                above += n[i];
            }
            found = __reduce_max_sync(0xffffffffu, found);
            const int bin = (int)(found & 511u) - 1;
            const unsigned take = (found >> 9) & 0x3FFFFFu;
            const bool whole = found >> 31;
            /* The upper words of the bin, and where its keys are when they have to be ranked. */
            unsigned most = 0, least = 0;
            each([&](int i, int j, uint32_t w) {
                const bool in = (WORDS > 0 ? bins[i] : bin_at(w)) == bin;
                most = in && w > most ? w : most;
                least = in && ~w > least ? ~w : least;
                if (in && !whole) {
                    const unsigned at = atomicAdd(&sc.found, 1u);
                    if (at < 32u) sc.candidates[at] = j;
                }
            });
            __syncwarp();
            t.most(most, least);
            bar = whole ? ~least - 1u : most;
            t.sync();
            const unsigned in_bin = whole ? 0u : sc.found;
            if (!whole && in_bin <= 32u) {
                if (t.me == 0) {
                    const int j = lane < (int)in_bin ? sc.candidates[lane] : -1;
                    const unsigned long long k = j >= 0 ? keys[j] : 0ull;
                    unsigned ahead = 0;
                    for (int c = 0; c < (int)in_bin; c++) {
                        const unsigned long long k2 = __shfl_sync(0xffffffffu, k, c);
                        const int j2 = __shfl_sync(0xffffffffu, j, c);
                        ahead += k2 > k || (k2 == k && j2 < j);
                    }
                    __syncwarp();
                    if (j >= 0 && ahead < take) keys[j] = ~0ull;
                    __syncwarp();
                }
                t.sync();
            } else if (!whole) {
                /* Keys of the bin: the largest value that `take` of them reach, three thresholds a step (two bits). */
                unsigned long long lo = (unsigned long long)~least << 32, hi = (unsigned long long)most << 32 | 0xFFFFFFFFull;
                while (lo < hi) {
                    const unsigned long long q = (hi - lo) / 4 + 1;     /* lo < t1 <= t2 <= t3 <= hi */
                    const unsigned long long t1 = lo + q, t2 = hi - t1 < q ? hi : t1 + q, t3 = hi - t2 < q ? hi : t2 + q;
                    unsigned n12 = 0, n3 = 0;
                    for (int j = j0 + lane; j < j1; j += 32) {
                        const unsigned long long k = keys[j];
                        if ((uint32_t)(k >> 32) > most) continue;
                        n12 += (unsigned)(k >= t1) + ((unsigned)(k >= t2) << 16);
                        n3 += k >= t3;
                    }
                    t.sum(n12, n3, x, y);
                    const unsigned n1 = n12 & 0xffffu, n2 = n12 >> 16;
                    if (n3 >= take) {
                        lo = t3;
                    } else if (n2 >= take) {
                        lo = t2;
                        hi = t3 - 1ull;
                    } else if (n1 >= take) {
                        lo = t1;
                        hi = t2 - 1ull;
                    } else {
                        hi = t1 - 1ull;
                    }
                }
                /* Above the cut all, equal to it from the lowest index. */
                unsigned over = 0, equal = 0, over_before, equal_before;
                for (int j = j0 + lane; j < j1; j += 32) {
                    const unsigned long long k = keys[j];
                    over += k > lo && (uint32_t)(k >> 32) <= most;
                    equal += k == lo;
                }
                t.sum(over, equal, over_before, equal_before);
                unsigned equal_left = take - over;
                equal_left = equal_before < equal_left ? equal_left - equal_before : 0u;
                for (int j = j0; j < j1; j += 32) {
                    const unsigned long long k = j + lane < j1 ? keys[j + lane] : 0ull;
                    const unsigned eq = __ballot_sync(0xffffffffu, k == lo);
                    if ((k > lo && (uint32_t)(k >> 32) <= most) || (k == lo && __popc(eq & before) < equal_left)) keys[j + lane] = ~0ull;
                    equal_left -= __popc(eq) < equal_left ? __popc(eq) : equal_left;
                }
                __syncwarp();
            }
            /* The words of ranked keys have changed. */
            if (WORDS > 0 && !whole) {
#pragma unroll
                for (int i = 0; i < WORDS; i++) words[i] = j0 + 32 * i + lane < j1 ? high_of(keys + j0 + 32 * i + lane) : kOut;
            }
        }
    }
    /* Each warp writes the blocks of its run behind those of the warps before it. */
    unsigned done = 0, none = 0;
    if (t.warps > 1) {
        unsigned taken = 0;
        each([&](int, int, uint32_t w) { taken += w > bar; });
        t.sum(taken, none, done, y);
    }
    if (WORDS > 0) {
        unsigned m[WORDS > 0 ? WORDS : 1];
#pragma unroll
        for (int i = 0; i < WORDS; i++) m[i] = __ballot_sync(0xffffffffu, words[i] > bar);
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            if (words[i] > bar) list[done + __popc(m[i] & before)] = j0 + 32 * i + lane;
            done += __popc(m[i]);
        }
    } else {
        for (int j = j0; j < j1; j += 32) {
            const bool take = j + lane < j1 && high_of(keys + j + lane) > bar;
            const unsigned m = __ballot_sync(0xffffffffu, take);
            if (take) list[done + __popc(m & before)] = j + lane;
            done += __popc(m);
        }
    }
    for (unsigned i = want + t.me * 32 + lane; i < (unsigned)p.topk; i += t.warps * 32) list[i] = -1;
}

template <int HD>
__global__ void __launch_bounds__(kSelThreads, 2)
k_block_select(const __grid_constant__ Select p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ TeamScratch scratch[kSelWarps];
    /* The rows as operand fragments [tile][product][lane], then [own_rows][k_blocks] keys. */
    double *qf = reinterpret_cast<double *>(smem_raw);
    const int tiles = p.rows > 8 ? 2 : 1;
    unsigned long long *keys = reinterpret_cast<unsigned long long *>(qf + (size_t)tiles * p.steps * 32);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.ctas > 1 ? (int)sm100::cluster_cta_rank() : 0;
    const int g = blockIdx.y;
    const long long r0 = (long long)(blockIdx.x / (unsigned)p.ctas) * p.rows;
    /* Before a CTA's shared memory is written by others it has to have started: told here, asked before the first store. */
    if (p.ctas > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b0 = rank * p.slice, b1 = b0 + p.slice < p.k_blocks ? b0 + p.slice : p.k_blocks;
    auto block_at = [&](int j0) -> const float * {
        const int j = j0 + (lane >> 2);
        return j < b1 ? p.km + ((size_t)j * p.kv_heads + g) * p.head_dim : nullptr;
    };
    Block<HD> next;
    next.load(block_at(b0 + warp * 8), lane);
    int qb = 0, head = 0;
    /* Four consecutive dimensions of a row at a time: products 4 g .. 4 g + 3 of lane 4 (row mod 8) + quarter. */
    const int quads = p.steps;                       /* per row */
    for (int i = threadIdx.x; i < tiles * 8 * quads; i += kSelThreads) {
        const int row = i / quads, qd = i - row * quads, e = qd * 4;
        const bool ok = row < p.rows && row_of(p, g, r0 + row, &qb, &head);
        const float *src = p.qm + ((size_t)qb * p.heads + head) * p.head_dim + e;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (HD > 0) {
            if (ok) {
                const float4 f = *reinterpret_cast<const float4 *>(src);
                v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (ok && e + k < p.head_dim) v[k] = src[k];
        }
        double *dst = qf + (size_t)((row >> 3) * p.steps + (qd & ~3)) * 32 + (row & 7) * 4 + (qd & 3);
#pragma unroll
        for (int k = 0; k < 4; k++) dst[k * 32] = (double)v[k];
    }
    __syncthreads();
    if (p.ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int j0 = b0 + warp * 8; j0 < b1; j0 += kSelWarps * 8) {
        const Block<HD> k = next;
        next.load(block_at(j0 + kSelWarps * 8), lane);       /* under the products of this tile */
        double d[2][2];
        score_tile<HD>(p, qf, k, lane, tiles, d);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int j = j0 + (lane & 3) * 2 + i;
            if (j >= b1) continue;
            const bool ok = !p.counts || p.counts[j] > 0;
            const bool kept = j < p.keep_first || j >= p.k_blocks - p.keep_last;
            for (int m = 0; m < tiles; m++) {
                const int row = m * 8 + (lane >> 2);
                if (row >= p.rows) continue;
                const unsigned long long key = !ok ? 0ull : (kept ? ~0ull : key_of(d[m][i]));
                /* Row r is chosen by CTA r mod ctas, as its row r / ctas. */
                unsigned long long *dst = keys + (size_t)(row / p.ctas) * p.k_blocks + j;
                if (p.ctas == 1)
                    *dst = key;
                else
                    asm volatile("st.shared::cluster.u64 [%0], %1;"
                                 ::"r"(sm100::map_to_cta(sm100::smem_u32(dst), row % p.ctas)), "l"(key) : "memory");
            }
        }
    }
    __syncwarp();
    if (p.ctas > 1) sm100::cluster_sync_all();
    else __syncthreads();
    TeamScratch &sc = scratch[warp / p.team];
    Team t = {warp % p.team, p.team, 1 + warp / p.team, sc.counts, 0u};
    for (int r = warp / p.team; r < p.own_rows; r += kSelWarps / p.team) {
        const int row = r * p.ctas + rank;
        if (row < p.rows && row_of(p, g, r0 + row, &qb, &head)) {
            unsigned long long *mine = keys + (size_t)r * p.k_blocks;
            int *list = p.list + ((size_t)head * p.q_blocks + qb) * p.topk;
            const int words = ((p.k_blocks + p.team - 1) / p.team + 31) / 32;        /* of a lane */
            if (words <= 4)
                choose<4>(p, t, mine, sc, list);
            else if (words <= 8)
                choose<8>(p, t, mine, sc, list);
            else if (words <= 12)
                choose<12>(p, t, mine, sc, list);
            else if (words <= 16)
                choose<16>(p, t, mine, sc, list);
            else
                choose<0>(p, t, mine, sc, list);
        }
        __syncwarp();
        t.sync();
    }
}

static int g_select_ready = 0;
static int g_max_ctas = 8;

/* Sixteen CTAs are more than every device promises a cluster (4 rows of 8 key
 * heads over 2048 blocks: 12.4 us so, 13.8 us with eight). */
static bool wide_clusters() {
    auto allow = [](auto kernel) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
    };
    bool ok = allow(k_block_select<128>) && allow(k_block_select<64>) && allow(k_block_select<0>);
    if (ok) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(kMaxCtas);
        cfg.blockDim = dim3(kSelThreads);
        cfg.dynamicSmemBytes = kWideSmem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kMaxCtas;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int fit = 0;
        ok = cudaOccupancyMaxActiveClusters(&fit, k_block_select<128>, &cfg) == cudaSuccess && fit > 0;
    }
    if (!ok) (void)cudaGetLastError();           /* a refusal here is an answer, not an error */
    return ok;
}

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
        set_error(IRIS_B200_EUNSUPPORTED, op, "more than 23552 key blocks");
        return IRIS_B200_EUNSUPPORTED;
    }
    if (q_blocks > 0 && (!list || !q_means || (k_blocks > 0 && !k_means))) return bad(op, "bad argument");
    if (head_dim > kMaxHeadDim) {
        set_error(IRIS_B200_EUNSUPPORTED, op, "head_dim above 512");
        return IRIS_B200_EUNSUPPORTED;
    }
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
    p.steps = (head_dim + 15) / 16 * 4;
    if (!g_select_ready) {
        if (!cuda_ok(cudaFuncSetAttribute(k_block_select<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmem), op) ||
            !cuda_ok(cudaFuncSetAttribute(k_block_select<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmem), op) ||
            !cuda_ok(cudaFuncSetAttribute(k_block_select<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmem), op))
            return IRIS_B200_ECUDA;
        g_max_ctas = wide_clusters() ? kMaxCtas : 8;
        g_select_ready = 1;
    }
    /* Rows of a cluster: as many as there are, up to two score tiles, and as
     * fit in shared memory with their keys. The blocks are cut over a cluster while
     * that leaves SMs idle otherwise (two CTAs per SM), down to one tile of
     * eight blocks per warp. */
    const long long rows = (long long)q_blocks * p.group;
    p.rows = rows < kSelRows ? (int)rows : kSelRows;
    auto tiles_of = [&] { return (rows + p.rows - 1) / p.rows; };
    p.ctas = 1;
    auto smem_of = [&] {
        p.own_rows = (p.rows + p.ctas - 1) / p.ctas;
        return (size_t)(p.rows > 8 ? 2 : 1) * p.steps * 256 + (size_t)p.own_rows * k_blocks * 8;
    };
    while (p.ctas < g_max_ctas && tiles_of() * kv_heads * p.ctas * 2 <= 2LL * g.sm_count && k_blocks >= p.ctas * 2 * kSelWarps * 8)
        p.ctas *= 2;
    if (p.ctas > 8 && smem_of() > kWideSmem) p.ctas = 8;
    /* Fewer rows per cluster where CTAs are left: choosing for a row takes
     * longer than its scores. A row is not shared by so many warps that they
     * have less than two blocks a lane. (30 query blocks x 5 heads x 120
     * blocks: 16 rows of a CTA 11.0 us, eight 7.3, four 8.3; 5 x 20 heads x
     * 549 blocks, two rows 11.8 us, one 8.9; 8 x 8 heads x 222 blocks, eight
     * rows 9.9 us, four 7.7, two 7.4, one 8.5.) */
    auto team_of = [](int own) { return own >= kSelWarps ? 1 : own > 2 ? 2 : own > 1 ? 4 : 8; };
    while (p.rows > 1 && tiles_of() * kv_heads * p.ctas * 2 <= 2LL * g.sm_count) {
        const int half = (p.rows + 1) / 2, own = (half + p.ctas - 1) / p.ctas, team = team_of(own);
        if (own >= (p.rows + p.ctas - 1) / p.ctas || (team > 1 && k_blocks < 64 * team)) break;
        p.rows = half;
    }
    while (p.rows > 1 && smem_of() > kSelSmem) p.rows--;
    const size_t smem = smem_of();
    p.slice = ((k_blocks + p.ctas - 1) / p.ctas + 7) / 8 * 8;
    p.team = team_of(p.own_rows);
    const long long clusters = tiles_of();
    if (clusters * p.ctas > INT_MAX) return bad(op, "too many query blocks");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    configure(&cfg, attr, dim3((unsigned)(clusters * p.ctas), (unsigned)kv_heads), kSelThreads, smem);
    if (p.ctas > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)p.ctas;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    const bool aligned = aligned16(k_means) && aligned16(q_means);
    const cudaError_t err = cudaLaunchKernelEx(&cfg, aligned && head_dim == 128  ? k_block_select<128>
                                                     : aligned && head_dim == 64 ? k_block_select<64>
                                                                                 : k_block_select<0>, p);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}
