/*
 * Attention over lists of key blocks for sm_100a: TMA loads of the listed
 * blocks, tcgen05 MMAs accumulating in tensor memory, online softmax with one
 * thread per query row. head_dim 128.
 *
 * Work decomposition
 *   A CTA takes one tile of up to 128 rows of a query block of one head. Two
 *   CTAs share an SM (half of its tensor memory and shared memory each), so
 *   that the tensor pipe works for one while the other is in its softmax; the
 *   dense kernel pairs two tiles in one CTA instead, which needs both to walk
 *   the same keys. The CTAs are not persistent: there is no work list to keep
 *   between launches, and neighbouring CTAs take neighbouring tiles of one
 *   head, so that its K and V stay in L2. Where the tiles do not fill the
 *   device the list of a tile is cut over the CTAs of a cluster, which merge
 *   their results through distributed shared memory.
 *
 * Keys
 *   A key tile is 128 rows made of 128 / k_block listed blocks (or a piece of
 *   a longer block), each its own TMA box, so blocks may lie anywhere. The
 *   producer warp reads the list 32 entries at a time, skips what names no
 *   block or holds no valid key, and publishes with every tile one bit per
 *   key: zero for rows behind seq_k, masked rows and the rows of a last tile
 *   that no block filled. Their scores become -inf whatever K holds; their V
 *   rows are cleared in shared memory before the MMA, since a zero probability
 *   does not cancel a NaN.
 *
 * Warps (256 threads)
 *   0-3  softmax: thread r owns row r of S / P / O
 *   4    producer
 *   5    MMA issuer, owner of the TMEM allocation
 *   6-7  idle: they complete the warpgroup that gives registers to the first
 *
 * Tensor memory (256 columns): S [0, 128), O [128, 256); P (bf16) over the
 * front of S. MMA order: QK(0) PV(0) QK(1) PV(1) ...; each PV in two halves of
 * 64 keys as the softmax hands them over. The softmax is that of the dense
 * kernel: base 2, the reference value of a row moves only when its maximum
 * grows by more than 8, P rounded to bf16 for the MMA while the row sum keeps
 * fp32. A row without any key yields zeros.
 *
 * Every wait on a barrier is bounded as in the dense kernel; a CTA that gives
 * up still takes part in the cluster's barriers.
 */
#include "attn_tc.cuh"
#include "common.cuh"

#include <cuda.h>
#include <math.h>

#include "kernels.h"

namespace iris_b200 {
namespace attn_blocks {

using namespace sm100;

static constexpr int kThreads = 256;
static constexpr int kHeadDim = 128;
static constexpr int kTile = 128;                        /* query rows / keys of a tile */
static constexpr int kHalfBytes = 128 * 64 * 2;          /* one [128 x 64] bf16 swizzled operand half */
static constexpr int kTileBytes = 2 * kHalfBytes;
static constexpr int kSmemQ = 0;                         /* later: staging of the output rows */
static constexpr int kSmemK = kTileBytes;                /* K and V; later: a cluster's partial rows */
static constexpr int kSmemV = 2 * kTileBytes;
static constexpr int kSmemBar = 3 * kTileBytes;
static constexpr float kRescaleThreshold = 8.0f;
static constexpr int kRegsSoftmax = 184, kRegsOther = 72;    /* 128 * 184 + 128 * 72 = the launch's 256 * 128 */
static constexpr int kMaxParts = 8;
static constexpr unsigned long long kDrainNs = 100000000ull;      /* for work in flight, beyond the wait limit */
static constexpr int kMetaSlots = 4;
static constexpr uint32_t kSbo = 1024 / 16;              /* 8 rows of 128 B, in 16-byte units */
static constexpr uint32_t kVLbo = kHalfBytes / 16;       /* next 64 dims */
static constexpr uint32_t kIdescQK = idesc_bf16(128, 128);
static constexpr uint32_t kIdescPV = kIdescQK | (1u << 16);

enum {
    BAR_Q_FULL = 0,
    BAR_K_FULL, BAR_K_EMPTY, BAR_V_FULL, BAR_V_EMPTY,
    BAR_S_FULL,
    BAR_P_FULL,                         /* 2: halves of the key tile */
    BAR_O_DONE = BAR_P_FULL + 2,
    BAR_DRAIN,
    BAR_META,                           /* kMetaSlots */
    BAR_COUNT = BAR_META + kMetaSlots
};
static constexpr int kOffTmemPtr = BAR_COUNT * 8;
static constexpr int kOffAbort = kOffTmemPtr + 4;
static constexpr int kOffMeta = 128;                     /* kMetaSlots x 32 bytes */
static constexpr int kOffMl = 256;                       /* 128 x (maximum, sum) */
static constexpr int kSmemBytes = kSmemBar + kOffMl + 128 * 8;
static_assert(kOffAbort + 4 <= kOffMeta && kOffMeta + kMetaSlots * 32 <= kOffMl, "barrier block");

/* What the producer publishes with a key tile. */
struct Meta {
    uint32_t bits[4];                   /* valid keys */
    uint32_t state;                     /* 1: a tile, all keys valid; 2: a tile with invalid keys; 0: the end */
    uint32_t pad[3];
};

struct Params {
    uint16_t *out;
    int ldo;
    int seq_q, seq_k, heads, group;     /* query heads per key head */
    const int *key_mask;
    const int *list;
    int list_len, q_block, q_blocks, k_block, k_blocks;
    int tiles;                          /* query tiles of a query block */
    int unit, units, per_entry;         /* rows of a TMA box, boxes of a tile, boxes of a list entry */
    int parts, part_len;                /* CTAs of a cluster, list entries of each */
    float scale_log2;
    unsigned int *status;
    unsigned long long wait_ns;
};

/* The bounded wait of the dense kernel, except that it first looks at the clock
 * after 64 tries: reading it takes about a thousand cycles, which a wait that is
 * nearly over should not pay (16 896 rows x 32 heads over 64 blocks: 1210 us
 * with the clock read on entry, 1060 us so). */
__device__ __forceinline__ bool wait_bar(const Ctx &c, int idx, uint32_t parity, int site) {
    const uint32_t bar = c.bars + idx * 8;
    unsigned long long t0 = 0;
    for (uint32_t spin = 1;; spin++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (spin % 64u != 0) continue;
        if (*c.abort_flag) return false;
        if (t0 == 0) t0 = global_ns();
        if (global_ns() - t0 > c.wait_ns || spin > (1u << 26)) {
            give_up(c, site, parity);
            return false;
        }
    }
}

struct Tile {
    int head, q0, rows;                 /* first row and rows that exist */
    const int *list;
    int e0, e1;                         /* this CTA's entries */
};
__device__ __forceinline__ Tile tile_of(const Params &p, int rank) {
    Tile t;
    t.head = (int)blockIdx.y;
    const int in_head = p.parts > 1 ? (int)(blockIdx.x / (unsigned)p.parts) : (int)blockIdx.x;
    const int qb = p.tiles > 1 ? in_head / p.tiles : in_head, in_block = (in_head - qb * p.tiles) * kTile;
    t.q0 = qb * p.q_block + in_block;
    int rows = p.q_block - in_block < kTile ? p.q_block - in_block : kTile;
    if (p.seq_q - t.q0 < rows) rows = p.seq_q - t.q0;
    t.rows = rows;                      /* <= 0: behind the last row of a short last block */
    t.list = p.list + ((size_t)t.head * p.q_blocks + qb) * p.list_len;
    t.e0 = rank * p.part_len;
    t.e1 = t.e0 + p.part_len < p.list_len ? t.e0 + p.part_len : p.list_len;
    if (rows <= 0) t.e1 = t.e0;
    return t;
}

__device__ __forceinline__ void producer(const Ctx &c, const Params &p, const Tile &t, const CUtensorMap *mq, const CUtensorMap *mk,
                                         const CUtensorMap *mv, uint32_t smem, volatile Meta *meta, int lane) {
    const int qcol = t.head * kHeadDim, kcol = (t.head / p.group) * kHeadDim;
    int j = 0;                          /* tiles published */
    int loads_k = 0, loads_v = 0;       /* tiles whose K / V copies were started */
    /* Q and the first entries of the list are on their way before anything else. */
    int entry = t.e0 + lane < t.e1 ? t.list[t.e0 + lane] : -1;
    if (lane == 0 && t.e0 < t.e1) {
        mbar_expect_tx(c.bars + BAR_Q_FULL * 8, kTileBytes);
        for (int half = 0; half < 2; half++)
            tma_load_2d(smem + kSmemQ + half * kHalfBytes, mq, qcol + half * 64, t.q0, c.bars + BAR_Q_FULL * 8);
    }
    __syncwarp();
    int filled = 0;                     /* boxes of the tile being put together; lane u holds the first row of box u */
    int row_of_unit = 0;
    uint32_t key_bits = 0;              /* lane w: valid keys [32 w, 32 w + 32) of the tile */
    bool ok = true;

    /* Publish (and load) the tile at hand; the end of the list when it is empty. */
    auto emit = [&]() -> bool {
        const int n = filled;
        const uint32_t par = (uint32_t)(j - 1) & 1u;
        /* QK(j - 1) is done: K's buffer is free, and every reader is through with the tile record of four tiles ago. */
        if (j > 0 && !__all_sync(0xffffffffu, wait_bar(c, BAR_K_EMPTY, par, 400))) return false;
        volatile Meta *m = meta + (j & (kMetaSlots - 1));
        const bool whole = __all_sync(0xffffffffu, lane >= 4 || key_bits == 0xFFFFFFFFu);
        if (lane < 4) m->bits[lane] = key_bits;
        key_bits = 0;
        if (lane == 0) m->state = n == 0 ? 0u : whole ? 1u : 2u;
        __syncwarp();
        if (lane == 0) mbar_arrive(c.bars + (BAR_META + (j & (kMetaSlots - 1))) * 8);
        if (n == 0) return true;
        const uint32_t bytes = (uint32_t)(n * p.unit * 256);
        if (lane == 0) mbar_expect_tx(c.bars + BAR_K_FULL * 8, bytes);
        __syncwarp();
        if (lane < n)
            for (int half = 0; half < 2; half++)
                tma_load_2d(smem + kSmemK + half * kHalfBytes + lane * p.unit * 128, mk, kcol + half * 64, row_of_unit,
                            c.bars + BAR_K_FULL * 8);
        loads_k++;
        if (j > 0 && !__all_sync(0xffffffffu, wait_bar(c, BAR_V_EMPTY, par, 401))) return false;
        if (lane == 0) mbar_expect_tx(c.bars + BAR_V_FULL * 8, bytes);
        __syncwarp();
        if (lane < n)
            for (int half = 0; half < 2; half++)
                tma_load_2d(smem + kSmemV + half * kHalfBytes + lane * p.unit * 128, mv, kcol + half * 64, row_of_unit,
                            c.bars + BAR_V_FULL * 8);
        __syncwarp();
        loads_v++;
        j++;
        filled = 0;
        return true;
    };

    /* One box of rows joins the tile at hand, unless the mask leaves none of them. */
    auto add = [&](int row0) -> bool {
        uint32_t any = 0, bits = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int key = 32 * w + lane;
            bool valid = key < p.unit && row0 + key < p.seq_k;
            if (valid && p.key_mask) valid = p.key_mask[row0 + key] != 0;
            const uint32_t b = __ballot_sync(0xffffffffu, valid);
            any |= b;
            /* Word of the tile that these keys belong to (two boxes of 16 keys share one). */
            if (lane == (filled * p.unit >> 5) + w) bits = p.unit == 16 ? b << (16 * (filled & 1)) : b;
        }
        if (any == 0) return true;
        if (32 * lane < kTile) key_bits |= bits;
        if (lane == filled) row_of_unit = row0;
        return ++filled < p.units || emit();
    };

    for (int e = t.e0; ok && e < t.e1; e += 32) {
        if (e > t.e0) entry = e + lane < t.e1 ? t.list[e + lane] : -1;
        unsigned todo = __ballot_sync(0xffffffffu, entry >= 0 && entry < p.k_blocks);
        while (ok && todo) {
            const int src = __ffs(todo) - 1;
            todo &= todo - 1;
            const int row0 = __shfl_sync(0xffffffffu, entry, src) * p.k_block;     /* < seq_k */
            for (int s = 0; ok && s < p.per_entry && row0 + s * kTile < p.seq_k; s++) ok = add(row0 + s * kTile);
        }
    }
    if (ok && filled > 0) ok = emit();
    /* (Without any block nobody else waits for Q, whose place the epilogue uses.) */
    if (ok && j == 0 && t.e0 < t.e1) ok = __all_sync(0xffffffffu, wait_bar(c, BAR_Q_FULL, 0, 402));
    if (ok) ok = emit();
    if (*c.abort_flag) {
        /* Nobody may be consuming any more: wait (bounded by the limit again) for the copies still in flight. */
        const unsigned long long t0 = global_ns();
        auto drain = [&](int bar, int n) {
            while (n > 0 && !mbar_try_wait(c.bars + bar * 8, (uint32_t)(n - 1) & 1u) && global_ns() - t0 < c.wait_ns + kDrainNs) {}
        };
        drain(BAR_Q_FULL, t.e0 < t.e1);
        drain(BAR_K_FULL, loads_k);
        drain(BAR_V_FULL, loads_v);
    }
}

/* Rows of V whose key does not count, cleared: four keys per lane. */
__device__ __forceinline__ void clear_rows(unsigned char *v, const volatile Meta *m, int lane) {
#pragma unroll 1
    for (int w = 0; w < 4; w++) {
        if ((m->bits[w] >> lane) & 1u) continue;
        const int row = 32 * w + lane;
#pragma unroll 1
        for (int half = 0; half < 2; half++)
            for (int ch = 0; ch < 8; ch++)
                *reinterpret_cast<uint4 *>(v + half * kHalfBytes + row * 128 + ch * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; }

__device__ __forceinline__ void mma_issuer(const Ctx &c, uint32_t smem, unsigned char *smem_gen, uint32_t tmem,
                                           const volatile Meta *meta, int lane) {
    const uint32_t hi = (uint32_t)(make_desc(0, 0, kSbo) >> 32);
    const uint32_t lo_q = (uint32_t)make_desc(smem + kSmemQ, 1, 0), lo_k = (uint32_t)make_desc(smem + kSmemK, 1, 0);
    const uint32_t lo_v = (uint32_t)make_desc(smem + kSmemV, kVLbo, 0);
    const bool leader = elect_one();
    bool ok = true;

    auto wait_all = [&](int bar, uint32_t par, int site) -> bool {
        return __all_sync(0xffffffffu, wait_bar(c, bar, par, site));
    };
    auto state_of = [&](int j) -> uint32_t { return meta[j & (kMetaSlots - 1)].state; };
    auto issue_qk = [&]() {
#pragma unroll
        for (int ks = 0; ks < kHeadDim / 16; ks++) {
            const uint32_t off = ((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4;
            if (leader) mma_ss(tmem, desc64(lo_q + off, hi), desc64(lo_k + off, hi), kIdescQK, ks > 0);
        }
        if (leader) {
            tc_commit(c.bars + BAR_S_FULL * 8);
            tc_commit(c.bars + BAR_K_EMPTY * 8);
        }
    };

    ok = wait_all(BAR_META, 0, 410);
    bool more = ok && state_of(0) != 0u;
    if (more) {
        ok = wait_all(BAR_Q_FULL, 0, 411) && wait_all(BAR_K_FULL, 0, 412);
        tc_fence_after();
        if (ok) issue_qk();
    }
    for (int j = 0; ok && more; j++) {
        const uint32_t par = (uint32_t)j & 1u;
        if (!(ok = wait_all(BAR_V_FULL, par, 413))) break;
        if (state_of(j) == 2u) clear_rows(smem_gen + kSmemV, meta + (j & (kMetaSlots - 1)), lane);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (!(ok = wait_all(BAR_P_FULL + h, par, 414 + h))) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
                if (leader)
                    mma_ts(tmem + 128, tmem + h * 32 + ks * 8, desc64(lo_v + ((h * 64 + ks * 16) * 128 >> 4), hi), kIdescPV,
                           j > 0 || h > 0 || ks > 0);
        }
        if (!ok) break;
        if (leader) tc_commit(c.bars + BAR_V_EMPTY * 8);
        const int nx = j + 1;
        if (!(ok = wait_all(BAR_META + (nx & (kMetaSlots - 1)), (uint32_t)(nx / kMetaSlots) & 1u, 416))) break;
        more = state_of(nx) != 0u;
        if (!more) {
            if (leader) tc_commit(c.bars + BAR_O_DONE * 8);
            break;
        }
        if (!(ok = wait_all(BAR_K_FULL, (uint32_t)nx & 1u, 417))) break;
        tc_fence_after();
        issue_qk();
    }
    if (!ok) {
        /* Let what was issued finish before the tensor memory goes away. */
        if (leader) tc_commit(c.bars + BAR_DRAIN * 8);
        const uint32_t bar = c.bars + BAR_DRAIN * 8;
        const unsigned long long t0 = global_ns();
        while (!mbar_try_wait(bar, 0) && global_ns() - t0 < c.wait_ns + kDrainNs) {}
    }
}

/* The row's running state after all its keys. */
struct RowState {
    float m, l;             /* reference (scaled log2 units) and sum */
    bool any;               /* O holds something */
    bool ok;
};

__device__ __forceinline__ RowState softmax_rows(const Ctx &c, const Params &p, const Tile &t, uint32_t tmem, const volatile Meta *meta) {
    const int row = threadIdx.x & 127;
    const uint32_t tS = tmem + ((uint32_t)(row & ~31) << 16), tO = tS + 128;
    const bool live = (row & ~31) < t.rows;              /* this warp has rows */
    const float sl2 = p.scale_log2;
    RowState st = {-INFINITY, 0.0f, false, true};
    for (int j = 0;; j++) {
        const int slot = j & (kMetaSlots - 1);
        if (!(st.ok = __all_sync(0xffffffffu, wait_bar(c, BAR_META + slot, (uint32_t)(j / kMetaSlots) & 1u, 420)))) return st;
        const uint32_t state = meta[slot].state;
        if (state == 0u) break;
        st.any = true;
        if (!(st.ok = __all_sync(0xffffffffu, wait_bar(c, BAR_S_FULL, (uint32_t)j & 1u, 421)))) return st;
        tc_fence_after();
        if (!live) {
            /* Rows that do not exist: whatever lies in P only meets rows of O that nobody reads. */
            tc_fence_before();
            mbar_arrive(c.bars + BAR_P_FULL * 8);
            mbar_arrive(c.bars + (BAR_P_FULL + 1) * 8);
            continue;
        }
        uint32_t s[128];
#pragma unroll
        for (int ch = 0; ch < 4; ch++) tmem_ld32(tS + ch * 32, s + ch * 32);
        tc_wait_ld();
        if (state == 2u) {
#pragma unroll
            for (int ch = 0; ch < 4; ch++) {
                const uint32_t bits = meta[slot].bits[ch];
                if (bits != 0xFFFFFFFFu) mask_chunk(s + ch * 32, bits);
            }
        }
        float mx8[8];
#pragma unroll
        for (int a = 0; a < 8; a++) mx8[a] = fmaxf(__uint_as_float(s[2 * a]), __uint_as_float(s[2 * a + 1]));
#pragma unroll
        for (int i = 16; i < 128; i += 16) {
#pragma unroll
            for (int a = 0; a < 8; a++)
                mx8[a] = max3(mx8[a], __uint_as_float(s[i + 2 * a]), __uint_as_float(s[i + 2 * a + 1]));
        }
        const float mx = fmaxf(max3(mx8[0], mx8[1], mx8[2]), max3(mx8[3], mx8[4], fmaxf(mx8[5], fmaxf(mx8[6], mx8[7]))));
        const float m_cand = fmaxf(st.m, mx * sl2);
        if (j == 0) {
            st.m = m_cand;
        } else {
            const bool need = m_cand > st.m + kRescaleThreshold;
            if (__any_sync(0xffffffffu, need)) {
                /* PV(j - 1) is complete (it was issued before the QK that filled S) and PV(j) waits for this warp. */
                const float alpha = need ? ex2(st.m - m_cand) : 1.0f;
                if (need) {
                    st.l *= alpha;
                    st.m = m_cand;
                }
#pragma unroll 1
                for (int i = 0; i < 4; i++) {
                    uint32_t o[32];
                    tmem_ld32(tO + i * 32, o);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    tmem_st32(tO + i * 32, o);
                }
            }
        }
        const float neg_ref = st.m == -INFINITY ? 0.0f : -st.m;
        float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            exp_half(s + 64 * h, sl2, neg_ref, sum4, tS + 32 * h);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(c.bars + (BAR_P_FULL + h) * 8);
        }
        st.l += (sum4[0] + sum4[2]) + (sum4[1] + sum4[3]);
    }
    if (st.any) {
        st.ok = __all_sync(0xffffffffu, wait_bar(c, BAR_O_DONE, 0, 422));
        tc_fence_after();
    }
    return st;
}

/* O times f -> bf16 rows, through 8 KB of staging per warp (two halves of 32
 * rows x 128 bytes, 16-byte chunks swizzled by the row): a thread owns a row,
 * memory wants eight threads per 128 bytes of it. */
__device__ __forceinline__ void store_rows(const Params &p, const Tile &t, uint32_t tmem, float f, bool any, unsigned char *stage) {
    const int row = threadIdx.x & 127, lane = threadIdx.x & 31, row0 = row & ~31;
    if (row0 >= t.rows) return;
    const uint32_t tO = tmem + ((uint32_t)row0 << 16) + 128;
    unsigned char *sw = stage + (row0 >> 5) * 8192;
    uint16_t *out = p.out + (size_t)(t.q0 + row0) * p.ldo + (size_t)t.head * kHeadDim;
    uint32_t o[128];
    if (any) {
#pragma unroll
        for (int q = 0; q < 4; q++) tmem_ld32(tO + q * 32, o + q * 32);
        tc_wait_ld();
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
#pragma unroll
        for (int ch = 0; ch < 8; ch++) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float a = __uint_as_float(o[64 * half + 8 * ch + 2 * e]), b = __uint_as_float(o[64 * half + 8 * ch + 2 * e + 1]);
                w[e] = any && f != 0.0f ? cvt_bf16x2(a * f, b * f) : 0u;
            }
            *reinterpret_cast<uint4 *>(sw + half * 4096 + lane * 128 + ((ch ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __syncwarp();
    const int ch = lane & 7;
#pragma unroll
    for (int half = 0; half < 2; half++) {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int r = k * 4 + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4 *>(sw + half * 4096 + r * 128 + ((ch ^ (r & 7)) << 4));
            if (row0 + r < t.rows) *reinterpret_cast<uint4 *>(out + (size_t)r * p.ldo + half * 64 + ch * 8) = v;
        }
    }
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
/* Address of 16-byte chunk ch (four columns) of a partial row: swizzled, so that rows do not share banks. */
__device__ __forceinline__ uint32_t part_addr(uint32_t smem, int row, int ch) {
    return smem + kSmemK + (uint32_t)row * 512u + (uint32_t)((ch ^ (row & 7)) << 4);
}

__global__ void __launch_bounds__(kThreads, 2)
k_attention_blocks_sm100(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                         const __grid_constant__ CUtensorMap tmv, const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) unsigned char smem_gen[];
    const uint32_t smem = smem_u32(smem_gen);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.parts > 1 ? (int)cluster_cta_rank() : 0;

    Ctx c;
    c.bars = smem + kSmemBar;
    c.abort_flag = reinterpret_cast<volatile uint32_t *>(smem_gen + kSmemBar + kOffAbort);
    c.status = p.status;
    c.wait_ns = p.wait_ns;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + kSmemBar + kOffTmemPtr);
    volatile Meta *meta = reinterpret_cast<volatile Meta *>(smem_gen + kSmemBar + kOffMeta);
    const Tile t = tile_of(p, rank);
    /* The producer sets up the barriers and starts at once; it only tells the
     * other warps, which wait here for the barriers and the tensor memory. The
     * launch is stream-serialised by program: nothing may be read or written
     * before the kernel ahead is complete, and no bounded wait may have begun.
     * (What is read may be written until then: no load through the
     * non-coherent path, which takes memory as constant for the whole kernel.) */
    uint32_t tmem = 0;
    if (warp == 4) {
        if (lane == 0) {
            for (int b = 0; b < BAR_COUNT; b++) mbar_init(c.bars + b * 8, b == BAR_P_FULL || b == BAR_P_FULL + 1 ? 128 : 1);
            *c.abort_flag = 0u;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        asm volatile("barrier.cta.arrive.aligned 1, %0;" ::"n"(kThreads) : "memory");
    } else {
        if (warp == 5) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem + kSmemBar + kOffTmemPtr), "r"(256u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
            tc_fence_before();
        }
        asm volatile("barrier.cta.sync.aligned 1, %0;" ::"n"(kThreads) : "memory");
        tc_fence_after();
        tmem = *tmem_slot;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");

    RowState st = {-INFINITY, 0.0f, false, true};
    if (warp < 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        st = softmax_rows(c, p, t, tmem, meta);
        if (p.parts == 1 && st.ok) store_rows(p, t, tmem, st.l != 0.0f ? 1.0f / st.l : 0.0f, st.any, smem_gen + kSmemQ);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == 4) producer(c, p, t, &tmq, &tmk, &tmv, smem, meta, lane);
        if (warp == 5) mma_issuer(c, smem, smem_gen, tmem, meta, lane);
        __syncwarp();
    }

    if (p.parts > 1) {
        /* The parts of a list meet: every CTA publishes the maxima and sums of
         * its rows, scales its rows by their share of the whole and leaves them
         * in shared memory; CTA r adds the columns [r, r + 1) * 128 / parts of
         * all of them. A row that no CTA has a key for stays zero. */
        const int row = threadIdx.x & 127;
        float2 *ml = reinterpret_cast<float2 *>(smem_gen + kSmemBar + kOffMl);
        if (warp < 4) ml[row] = make_float2(st.m, st.l);
        cluster_sync_all();
        if (warp < 4 && (row & ~31) < t.rows) {
            float m = -INFINITY, l = 0.0f;
            for (int r = 0; r < p.parts; r++) m = fmaxf(m, ld_cluster_f2(map_to_cta(smem + kSmemBar + kOffMl + row * 8, r)).x);
            for (int r = 0; r < p.parts; r++) {
                const float2 o = ld_cluster_f2(map_to_cta(smem + kSmemBar + kOffMl + row * 8, r));
                if (o.y != 0.0f) l += o.y * ex2(o.x - m);
            }
            const float f = st.ok && st.any && st.l != 0.0f ? ex2(st.m - m) / l : 0.0f;
            const uint32_t tO = tmem + ((uint32_t)(row & ~31) << 16) + 128;
#pragma unroll 1
            for (int q = 0; q < 4; q++) {
                uint32_t o[32];
                if (st.any) {
                    tmem_ld32(tO + q * 32, o);
                    tc_wait_ld();
                }
#pragma unroll
                for (int ch = 0; ch < 8; ch++) {
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (f != 0.0f)
                        v = make_float4(__uint_as_float(o[4 * ch]) * f, __uint_as_float(o[4 * ch + 1]) * f,
                                        __uint_as_float(o[4 * ch + 2]) * f, __uint_as_float(o[4 * ch + 3]) * f);
                    if (row < t.rows)
                        *reinterpret_cast<float4 *>(smem_gen + (part_addr(smem, row, q * 8 + ch) - smem)) = v;
                }
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (warp < 4) {
            const int width = kHeadDim / p.parts, chunks = width / 8;
            for (int i = threadIdx.x; i < t.rows * chunks; i += 128) {
                const int r = i / chunks, col = rank * width + (i - r * chunks) * 8;
                float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                for (int other = 0; other < p.parts; other++) {
                    const float4 a = ld_cluster_f4(map_to_cta(part_addr(smem, r, col / 4), other));
                    const float4 b = ld_cluster_f4(map_to_cta(part_addr(smem, r, col / 4 + 1), other));
                    s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
                    s[4] += b.x; s[5] += b.y; s[6] += b.z; s[7] += b.w;
                }
                if (st.ok)
                    *reinterpret_cast<uint4 *>(p.out + (size_t)(t.q0 + r) * p.ldo + (size_t)t.head * kHeadDim + col) =
                        make_uint4(cvt_bf16x2(s[0], s[1]), cvt_bf16x2(s[2], s[3]), cvt_bf16x2(s[4], s[5]), cvt_bf16x2(s[6], s[7]));
            }
        }
        __syncwarp();
        cluster_sync_all();             /* nobody leaves while its rows are being read */
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
    }
}

/* CTAs that share the list of a query tile. With fewer tiles than the device
 * has room for (two CTAs per SM) the lists are cut, down to two key tiles per
 * CTA. (More tiles than that gain nothing: 306 tiles of 30 key tiles 117 us
 * whole, 122 us in two parts.) */
static int choose_parts(long long items, long long key_tiles, int sms) {
    int parts = 1;
    while (parts < kMaxParts && items * parts * 2 <= 2LL * sms && key_tiles >= 4 * parts) parts *= 2;
    return parts;
}

static int g_ready = 0;

}  // namespace attn_blocks

void attention_blocks_release(void) { attn_blocks::g_ready = 0; }

bool attention_blocks_sm100_supported(const BlockAttnArgs &a) {
    const uintptr_t bits = (uintptr_t)a.out | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
    const long long tiles = (long long)a.heads * a.q_blocks * (((a.q_block < a.seq_q ? a.q_block : a.seq_q) + 127) / 128);
    return a.head_dim == attn_blocks::kHeadDim && (a.k_block == 16 || a.k_block == 32 || a.k_block == 64 || a.k_block % 128 == 0) &&
           a.ldo % 8 == 0 && a.ldq % 8 == 0 && a.ldk % 8 == 0 && a.ldv % 8 == 0 && (bits & 15) == 0 && a.seq_k > 0 &&
           tiles <= 0x7FFFFFFFll / attn_blocks::kMaxParts;
}

int launch_attention_blocks_sm100(const BlockAttnArgs &a) {
    using namespace attn_blocks;
    const char *op = "attention_blocks";
    if (!g_ready) {
        if (!cuda_ok(cudaFuncSetAttribute(k_attention_blocks_sm100, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes), op))
            return IRIS_B200_ECUDA;
        g_ready = 1;
    }
    Params p = {};
    p.out = a.out;
    p.ldo = a.ldo;
    p.seq_q = a.seq_q;
    p.seq_k = a.seq_k;
    p.heads = a.heads;
    p.group = a.heads / a.kv_heads;
    p.key_mask = a.key_mask;
    p.list = a.list;
    p.list_len = a.list_len;
    p.q_block = a.q_block < a.seq_q ? a.q_block : a.seq_q;
    p.q_blocks = a.q_blocks;
    p.k_block = a.k_block;
    p.k_blocks = a.k_blocks;
    p.tiles = (p.q_block + kTile - 1) / kTile;
    p.unit = a.k_block < kTile ? a.k_block : kTile;
    p.units = kTile / p.unit;
    p.per_entry = a.k_block < kTile ? 1 : a.k_block / kTile;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.status = g.dev_status;
    p.wait_ns = wait_limit_ns();
    const long long items = (long long)a.heads * a.q_blocks * p.tiles;
    const long long key_tiles = ((long long)a.list_len * p.per_entry + p.units - 1) / p.units;
    p.parts = choose_parts(items, key_tiles, g.sm_count);
    /* Whole key tiles per part, where every entry names a block. */
    const int tile_entries = p.units > 1 ? p.units : 1;
    p.part_len = ((a.list_len + p.parts - 1) / p.parts + tile_entries - 1) / tile_entries * tile_entries;
    CUtensorMap tmq, tmk, tmv;
    if (!make_tensor_map(&tmq, a.q, a.seq_q, a.heads * kHeadDim, a.ldq, kTile) ||
        !make_tensor_map(&tmk, a.k, a.seq_k, a.kv_heads * kHeadDim, a.ldk, p.unit) ||
        !make_tensor_map(&tmv, a.v, a.seq_k, a.kv_heads * kHeadDim, a.ldv, p.unit))
        return IRIS_B200_ECUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.q_blocks * p.tiles * p.parts), (unsigned)a.heads);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
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
    const cudaError_t err = cudaLaunchKernelEx(&cfg, k_attention_blocks_sm100, tmq, tmk, tmv, p);
    g.launches++;
    return cuda_ok(err, op) ? IRIS_B200_OK : IRIS_B200_ECUDA;
}

}  // namespace iris_b200
