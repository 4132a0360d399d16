/*
 * Attention over lists of key blocks for sm_100a: TMA loads of the listed
 * blocks, tcgen05 MMAs accumulating in tensor memory, online softmax with one
 * thread per query row. head_dim 128.
 *
 * Work decomposition
 *   A CTA takes tiles of up to 128 rows of a query block of one head, one after
 *   the other. Two CTAs share an SM (half of its tensor memory and shared
 *   memory each), so that the tensor pipe works for one while the other is in
 *   its softmax; the dense kernel pairs two tiles in one CTA instead, which
 *   needs both to walk the same keys. The tiles go round the CTAs in order:
 *   those in flight belong to few heads, whose K and V stay in L2, and Q, the
 *   list, K and V of the next tile are on their way while the last one's
 *   softmax, product and store finish (4333 rows x 30 heads over 18 blocks of
 *   64 keys: 94 us with a CTA per tile, 86 us so). Where the tiles do not fill
 *   the device the list of a tile is cut over the CTAs of a cluster, which
 *   merge their results through distributed shared memory.
 *
 * Keys
 *   A key tile is 128 rows made of 128 / k_block listed blocks (or a piece of
 *   a longer block), each its own TMA box, so blocks may lie anywhere. The
 *   producer warp reads the list 32 entries at a time, skips what names no
 *   block or holds no valid key, and publishes with every tile one bit per
 *   key: zero for rows behind seq_k, masked rows and the rows of a last tile
 *   that no block filled. Their scores become -inf whatever K holds; their V
 *   rows are cleared in shared memory before the MMA, since a zero probability
 *   does not cancel a NaN. The mask is read one key tile ahead.
 *
 * Warps (256 threads)
 *   0-3      softmax: thread r owns row r of S / P / O
 *   4 or 6   producer (6 in the second half of the CTAs, so that the two on an
 *            SM, one of either half, do not share a scheduler)
 *   5 or 7   MMA issuer, owner of the TMEM allocation
 *   others   idle: they complete the warpgroup that gives registers to the first
 *
 * Tensor memory (256 columns): S [0, 128), O [128, 256); P (bf16) over the
 * front of S. MMA order: QK(0) PV(0) QK(1) PV(1) ...; each PV in two halves of
 * 64 keys as the softmax hands them over. The softmax is that of the dense
 * kernel: base 2, the reference value of a row moves only when its maximum
 * grows by more than 8. P is rounded to bf16, since the operands of one
 * kind::f16 product have one type and V is bf16; the row sum keeps fp32. That
 * rounding is 0.0016 of a result (root mean square of a bf16 rounding over a
 * mantissa) beside the 0.0017 of the result's own: together 0.0023 against 64
 * bits, and more bits would take a second product. A row without any key yields
 * zeros.
 *
 * Records: the producer hands the tiles of keys and the end of every query
 * tile to the softmax and MMA warps through a ring of four records, which all
 * of them free again. Buffers of Q, K, V, S / P and O are single; barrier
 * parities count key tiles (Q, O: query tiles with keys) of the whole CTA.
 *
 * Bound by the chain scores -> softmax -> product: 16 896 rows x 32 heads over
 * 64 blocks of 64 keys take 1 020 to 1 030 us in a short run (1.10 to 1.11
 * PFLOP/s) and 1 180 in a run of seconds, at 1 600 MHz under the 1000 W cap, where
 * the products alone would take 690 and 810 at the burst and the sustained rate;
 * tensor pipe and exponential unit are busy for 55 % of the cycles. Per pair of key tiles an SM spends about 3 700
 * cycles, 2 048 of them in products and, beside them, 2 048 in exponentials;
 * the two CTAs alternate, a softmax takes 1 700 cycles and the way from its
 * last probability to its next scores 1 400.
 *
 * Every wait on a barrier is bounded as in the dense kernel; a CTA that gives
 * up still takes part in the cluster's barriers, and before it leaves it waits
 * (bounded again) for its copies and products in flight.
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
static constexpr int kSmemQ = 0;
static constexpr int kSmemK = kTileBytes;                /* K and V; later: a cluster's partial rows */
static constexpr int kSmemV = 2 * kTileBytes;
static constexpr int kSmemStage = 3 * kTileBytes;        /* output rows, 4 KB per softmax warp; or a cluster's (maximum, sum) */
static constexpr int kSmemBar = kSmemStage + 4 * 4096;
static constexpr float kRescaleThreshold = 8.0f;
static constexpr int kRegsSoftmax = 184, kRegsOther = 72;    /* 128 * 184 + 128 * 72 = the launch's 256 * 128 */
static constexpr int kMaxParts = 8;
static constexpr unsigned long long kDrainNs = 100000000ull;      /* for work in flight, beyond the wait limit */
static constexpr int kMetaSlots = 4;
static constexpr uint32_t kReadsPerBeat = 8192;
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
    BAR_META,                           /* kMetaSlots: a record is there */
    BAR_META_FREE = BAR_META + kMetaSlots,      /* kMetaSlots: its readers, four softmax warps and the MMA warp, are through */
    BAR_COUNT = BAR_META_FREE + kMetaSlots
};
static constexpr int kOffTmemPtr = BAR_COUNT * 8;
static constexpr int kOffAbort = kOffTmemPtr + 4;
static constexpr int kOffBeat = kOffAbort + 4;           /* grows while the producer reads on */
static constexpr int kOffMeta = 160;                     /* kMetaSlots x 32 bytes */
static constexpr int kSmemBytes = kSmemBar + kOffMeta + kMetaSlots * 32;
static_assert(kOffBeat + 4 <= kOffMeta, "barrier block");
static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");

/* What the producer publishes: the key tiles of a query tile, and its end. */
static constexpr uint32_t kEnd = 0, kEndUnused = 4;      /* unused: Q was loaded, but there was no key tile */
static constexpr uint32_t kWhole = 1, kPartly = 2;       /* a key tile with all keys valid, with invalid keys */
__device__ __forceinline__ bool is_end(uint32_t state) { return (state & 3u) == kEnd; }

struct Meta {
    uint32_t bits[4];                   /* valid keys */
    uint32_t state;                     /* kEnd, kEndUnused, kWhole or kPartly */
    uint32_t pad[3];
};

struct Params {
    uint16_t *out;
    int ldo;
    int seq_q, seq_k, heads, group;     /* query heads per key head */
    const int *key_mask;
    const int *list;
    int list_len, q_block, q_blocks, k_block, k_blocks;
    int tiles, per_head, items;         /* query tiles of a query block, of a head, of the launch */
    int unit, unit_log, units, per_entry;       /* rows of a TMA box, boxes of a tile, boxes of a list entry */
    int parts, part_len;                /* CTAs of a cluster, list entries of each */
    float scale_log2;
    unsigned int *status;
    unsigned long long wait_ns;
};

/* The bounded wait of the dense kernel, except that it first looks at the clock
 * after 64 tries: reading it takes about a thousand cycles, which a wait that is
 * nearly over should not pay (16 896 rows x 32 heads over 64 blocks: 1210 us
 * with the clock read on entry, 1060 us so).
 * A record may be millions of list entries away. The MMA warp's wait for one
 * (kReader) begins anew while the producer shows that it reads on, and the
 * softmax warps (kFollower), which wait for the same record, leave the clock to
 * the MMA warp: they see its flag. */
enum WaitKind { kPlain, kReader, kFollower };
template <WaitKind KIND = kPlain>
__device__ __forceinline__ bool wait_bar(const Ctx &c, int idx, uint32_t parity, int site) {
    const uint32_t bar = c.bars + idx * 8;
    unsigned long long t0 = 0;
    uint32_t beat = 0;
    for (uint32_t spin = 1;; spin++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (spin % 64u != 0) continue;
        if (*c.abort_flag) return false;
        if (spin <= (1u << 26)) {
            if (KIND == kFollower) continue;
            if (t0 == 0) t0 = global_ns();
            if (global_ns() - t0 <= c.wait_ns) continue;
            if (KIND == kReader && c.abort_flag[1] != beat) {
                beat = c.abort_flag[1];
                t0 = 0;
                spin = 0;
                continue;
            }
        }
        give_up(c, site, parity);
        return false;
    }
}

struct Tile {
    int head, q0, rows;                 /* first row and rows that exist */
    const int *list;
    int e0, e1;                         /* this CTA's entries */
};
__device__ __forceinline__ Tile tile_of(const Params &p, int item, int rank) {
    Tile t;
    t.head = item / p.per_head;
    const int in_head = item - t.head * p.per_head;
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
/* A CTA's query tiles: first_item, + item_step, ... below p.items. (A cluster has one.) */
__device__ __forceinline__ int first_item(const Params &p) { return p.parts > 1 ? (int)(blockIdx.x / (unsigned)p.parts) : (int)blockIdx.x; }
__device__ __forceinline__ int item_step(const Params &p) { return p.parts > 1 ? p.items : (int)gridDim.x; }

/* How many loads of Q, K and V a producer has issued. */
struct Loads {
    int q, k, v;
};

/* What has to have happened before the shared memory goes away, looked at
 * behind the CTA's last barrier. The tensor cores have arrived for the last
 * products with K and V (the softmax warps saw their end by a barrier of a later
 * commit, which does not order the arrivals); in a CTA that gave up, where nobody
 * may have waited for the last loads, those are in (bounded by the limit again). */
__device__ __forceinline__ void settle_loads(const Ctx &c, const Loads &n) {
    if (!*c.abort_flag) {
        const uint32_t par = (uint32_t)(n.k - 1) & 1u;
        if (n.k > 0 && wait_bar(c, BAR_K_EMPTY, par, 405)) wait_bar(c, BAR_V_EMPTY, par, 406);
        return;
    }
    const unsigned long long t0 = global_ns();
    auto drain = [&](int bar, int loads) {
        while (loads > 0 && !mbar_try_wait(c.bars + bar * 8, (uint32_t)(loads - 1) & 1u) && global_ns() - t0 < c.wait_ns + kDrainNs) {}
    };
    drain(BAR_Q_FULL, n.q);
    drain(BAR_K_FULL, n.k);
    drain(BAR_V_FULL, n.v);
}

__device__ __forceinline__ Loads producer(const Ctx &c, const Params &p, int rank, const CUtensorMap *mq, const CUtensorMap *mk,
                                          const CUtensorMap *mv, uint32_t smem, volatile Meta *meta, int lane) {
    int r = 0, j = 0;                   /* records published, key tiles loaded */
    int loads_q = 0, loads_v = 0;
    int filled = 0;                     /* boxes of the key tile being put together; lane u holds the first row of box u */
    int row_of_unit = 0;
    uint32_t key_bits = 0;              /* lane w: valid keys [32 w, 32 w + 32) of the tile */
    bool ok = true, unused = false;     /* unused: Q is loaded, no key tile of it yet */
    int kcol = 0;

    auto load_q = [&](const Tile &t) {
        unused = t.e0 < t.e1;
        if (!unused) return;
        if (lane == 0) {
            mbar_expect_tx(c.bars + BAR_Q_FULL * 8, kTileBytes);
            for (int half = 0; half < 2; half++)
                tma_load_2d(smem + kSmemQ + half * kHalfBytes, mq, t.head * kHeadDim + half * 64, t.q0, c.bars + BAR_Q_FULL * 8);
        }
        __syncwarp();
        loads_q++;
    };

    /* Publish (and load) the key tile at hand, or the end of the query tile. */
    auto emit = [&](bool end) -> bool {
        const int slot = r & (kMetaSlots - 1);
        if (r >= kMetaSlots && !__all_sync(0xffffffffu, wait_bar(c, BAR_META_FREE + slot, (uint32_t)(r / kMetaSlots - 1) & 1u, 403)))
            return false;
        volatile Meta *m = meta + slot;
        const bool whole = __all_sync(0xffffffffu, lane >= 4 || key_bits == 0xFFFFFFFFu);
        if (lane < 4) m->bits[lane] = key_bits;
        key_bits = 0;
        if (lane == 0) m->state = end ? (unused ? kEndUnused : kEnd) : whole ? kWhole : kPartly;
        __syncwarp();
        if (lane == 0) mbar_arrive(c.bars + (BAR_META + slot) * 8);
        r++;
        if (end) return true;
        const int n = filled;
        const uint32_t bytes = (uint32_t)(n * p.unit * 256), par = (uint32_t)(j - 1) & 1u;
        if (j > 0 && !__all_sync(0xffffffffu, wait_bar(c, BAR_K_EMPTY, par, 400))) return false;       /* QK(j - 1) is done */
        if (lane == 0) mbar_expect_tx(c.bars + BAR_K_FULL * 8, bytes);
        unused = false;
        __syncwarp();
        if (lane < n)
            for (int half = 0; half < 2; half++)
                tma_load_2d(smem + kSmemK + half * kHalfBytes + lane * p.unit * 128, mk, kcol + half * 64, row_of_unit,
                            c.bars + BAR_K_FULL * 8);
        __syncwarp();
        j++;
        filled = 0;
        if (j > 1 && !__all_sync(0xffffffffu, wait_bar(c, BAR_V_EMPTY, par, 401))) return false;
        if (lane == 0) mbar_expect_tx(c.bars + BAR_V_FULL * 8, bytes);
        __syncwarp();
        if (lane < n)
            for (int half = 0; half < 2; half++)
                tma_load_2d(smem + kSmemV + half * kHalfBytes + lane * p.unit * 128, mv, kcol + half * 64, row_of_unit,
                            c.bars + BAR_V_FULL * 8);
        __syncwarp();
        loads_v++;
        return true;
    };

    /* A sign of life (and a look at the others') every so many reads without a key tile, each the latency of a load: milliseconds. */
    uint32_t reads = 0;
    auto read_on = [&]() -> bool {
        if (++reads % kReadsPerBeat != 0) return true;
        if (lane == 0) c.abort_flag[1] = reads;
        return __all_sync(0xffffffffu, *c.abort_flag == 0u);
    };

    /* The next boxes of a window of 32 entries, a tile's number of them at most: lane u gets the first row of box u, -1 behind the last. */
    unsigned todo = 0;
    int sub = 0;                        /* box of a long block */
    auto take = [&](int entry) -> int {
        int row = -1;
        if (p.per_entry == 1) {
            for (int n = 0; todo && n < p.units; n++) {
                const int v = __shfl_sync(0xffffffffu, entry, __ffs(todo) - 1) * p.k_block;     /* < seq_k */
                todo &= todo - 1;
                if (lane == n) row = v;
            }
        } else if (todo) {
            const int v = __shfl_sync(0xffffffffu, entry, __ffs(todo) - 1) * p.k_block + sub * kTile;
            if (lane == 0) row = v;
            if (++sub == p.per_entry || v >= p.seq_k - kTile) {
                sub = 0;
                todo &= todo - 1;
            }
        }
        return row;
    };
    /* What the mask says of their keys: keys 32 w + lane of the boxes side by side. Only looked at one step later. */
    auto fetch = [&](int row, int flag[4]) {
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int key = 32 * w + lane, r0 = __shfl_sync(0xffffffffu, row, key >> p.unit_log), k = r0 + (key & (p.unit - 1));
            flag[w] = 0;
            if (r0 >= 0 && k < p.seq_k) flag[w] = p.key_mask ? p.key_mask[k] : 1;
        }
    };
    /* The boxes join the key tile at hand, except those of which the mask leaves nothing. */
    auto add = [&](int row, int flag[4]) -> bool {
        if (!p.key_mask && filled == 0 && __all_sync(0xffffffffu, lane >= p.units || (row >= 0 && row <= p.seq_k - p.unit))) {
            key_bits = 0xFFFFFFFFu;
            row_of_unit = row;
            filled = p.units;
            return emit(false);
        }
        uint32_t word = 0;              /* lane w < 4: keys [32 w, 32 w + 32) */
        if (!p.key_mask) fetch(row, flag);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const uint32_t b = __ballot_sync(0xffffffffu, flag[w] != 0);
            if (lane == w) word = b;
        }
        const bool some = p.unit == 16 ? (word & 0xFFFFu) && (word >> 16) : word != 0;
        if (filled == 0 && __all_sync(0xffffffffu, lane >= 4 || some)) {
            key_bits = word;
            row_of_unit = row;
            filled = p.units;
            return emit(false);
        }
        const int words = p.unit >> 5;                          /* of a box; 0: half a word */
        for (int u = 0; u < p.units; u++) {
            const int r0 = __shfl_sync(0xffffffffu, row, u);
            if (r0 < 0) break;
            if (words == 0) {
                const uint32_t half = (__shfl_sync(0xffffffffu, word, u >> 1) >> (16 * (u & 1))) & 0xFFFFu;
                if (half == 0) continue;
                if (lane == filled >> 1) key_bits |= half << (16 * (filled & 1));
            } else {
                const int at = lane - filled * words;           /* word of the box that this lane keeps */
                const uint32_t v = __shfl_sync(0xffffffffu, word, (u * words + at) & 31);
                const bool mine = at >= 0 && at < words;
                if (!__any_sync(0xffffffffu, mine && v != 0)) continue;
                if (mine) key_bits = v;
            }
            if (lane == filled) row_of_unit = r0;
            if (++filled == p.units && !emit(false)) return false;
        }
        return read_on();
    };

    const int step = item_step(p);
    int item = first_item(p);
    Tile t = tile_of(p, item, rank);
    int entry = t.e0 + lane < t.e1 ? t.list[t.e0 + lane] : -1;
    load_q(t);
    while (ok) {
        kcol = (t.head / p.group) * kHeadDim;
        /* The first entries of the next query tile are on their way meanwhile. */
        const int next_item = item < p.items - step ? item + step : -1;
        Tile t2 = t;
        int entry2 = -1;
        if (next_item >= 0) {
            t2 = tile_of(p, next_item, rank);
            if (t2.e0 + lane < t2.e1) entry2 = t2.list[t2.e0 + lane];
        }
        for (int e = t.e0; ok && e < t.e1; e += 32) {
            if (e > t.e0) entry = e + lane < t.e1 ? t.list[e + lane] : -1;
            ok = read_on();
            todo = __ballot_sync(0xffffffffu, entry >= 0 && entry < p.k_blocks);
            int row = take(entry), flag[4], next_flag[4];
            if (p.key_mask) fetch(row, flag);
            while (ok && __any_sync(0xffffffffu, row >= 0)) {
                const int next_row = take(entry);
                if (p.key_mask) fetch(next_row, next_flag);
                ok = add(row, flag);
                row = next_row;
#pragma unroll
                for (int w = 0; w < 4; w++) flag[w] = next_flag[w];
            }
        }
        if (ok && filled > 0) ok = emit(false);
        if (ok) ok = emit(true);
        /* A Q that no product is made with has to arrive before the next one is asked for, and before the CTA
         * leaves: nobody else waits for it, and its shared memory may be another CTA's by then. */
        if (ok && unused) ok = __all_sync(0xffffffffu, wait_bar(c, BAR_Q_FULL, (uint32_t)(loads_q - 1) & 1u, 402));
        if (!ok || next_item < 0) break;
        /* The last product with Q is done. */
        if (!unused && j > 0) ok = __all_sync(0xffffffffu, wait_bar(c, BAR_K_EMPTY, (uint32_t)(j - 1) & 1u, 404));
        if (!ok) break;
        item = next_item;
        t = t2;
        entry = entry2;
        load_q(t);
    }
    return {loads_q, j, loads_v};
}

/* Rows of V whose key does not count, cleared: 32 rows side by side where none
 * of them does, else two at a time, half a warp each. */
__device__ __forceinline__ void clear_rows(unsigned char *v, const volatile Meta *m, int lane) {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    unsigned char *mine = v + ((lane >> 3) & 1) * kHalfBytes + (lane & 7) * 16;
#pragma unroll 1
    for (int w = 0; w < 4; w++) {
        uint32_t out = ~m->bits[w];
        if (out == 0xFFFFFFFFu) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                *reinterpret_cast<uint4 *>(v + (i >> 3) * kHalfBytes + w * 4096 + (i & 7) * 512 + lane * 16) = zero;
            continue;
        }
        while (out) {
            const int r0 = __ffs(out) - 1;
            out &= out - 1;
            const int r1 = out ? __ffs(out) - 1 : r0;
            out &= out - 1;
            *reinterpret_cast<uint4 *>(mine + (32 * w + (lane < 16 ? r0 : r1)) * 128) = zero;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; }

__device__ __forceinline__ void mma_issuer(const Ctx &c, const Params &p, uint32_t smem, unsigned char *smem_gen, uint32_t tmem,
                                           const volatile Meta *meta, int lane) {
    const uint32_t hi = (uint32_t)(make_desc(0, 0, kSbo) >> 32);
    const uint32_t lo_q = (uint32_t)make_desc(smem + kSmemQ, 1, 0), lo_k = (uint32_t)make_desc(smem + kSmemK, 1, 0);
    const uint32_t lo_v = (uint32_t)make_desc(smem + kSmemV, kVLbo, 0);
    const bool leader = elect_one();
    bool ok = true;

    auto wait_all = [&](int bar, uint32_t par, int site) -> bool {
        return __all_sync(0xffffffffu, wait_bar(c, bar, par, site));
    };
    auto release = [&](int record) {
        __syncwarp();
        if (lane == 0) mbar_arrive(c.bars + (BAR_META_FREE + (record & (kMetaSlots - 1))) * 8);
    };
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

    int r = 0, j = 0, nq = 0;           /* records, key tiles whose scores were issued, query tiles with any */
    for (int item = first_item(p); ok; item += item_step(p)) {
        bool some = false;
        while (ok) {
            const int slot = r & (kMetaSlots - 1);
            if (!(ok = __all_sync(0xffffffffu, wait_bar<kReader>(c, BAR_META + slot, (uint32_t)(r / kMetaSlots) & 1u, 410)))) break;
            const uint32_t state = meta[slot].state;
            if (is_end(state)) {
                if (some && leader) tc_commit(c.bars + BAR_O_DONE * 8);
                nq += state == kEndUnused;
                release(r++);
                break;
            }
            const uint32_t par = (uint32_t)j & 1u;
            if (!some && !(ok = wait_all(BAR_Q_FULL, (uint32_t)nq++ & 1u, 411))) break;
            if (!(ok = wait_all(BAR_K_FULL, par, 412))) break;
            tc_fence_after();
            issue_qk();
            if (!(ok = wait_all(BAR_V_FULL, par, 413))) break;
            if (state == kPartly) clear_rows(smem_gen + kSmemV, meta + slot, lane);
            release(r++);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (!(ok = wait_all(BAR_P_FULL + h, par, 414 + h))) break;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    if (leader)
                        mma_ts(tmem + 128, tmem + h * 32 + ks * 8, desc64(lo_v + ((h * 64 + ks * 16) * 128 >> 4), hi), kIdescPV,
                               some || h > 0 || ks > 0);
            }
            if (!ok) break;
            if (leader) tc_commit(c.bars + BAR_V_EMPTY * 8);
            some = true;
            j++;
        }
        if (item >= p.items - item_step(p)) break;
    }
}

/* In a CTA that gave up: the products issued so far (by the lane that the same election chose) end before their operands and
 * the tensor memory go away. */
__device__ __forceinline__ void drain_products(const Ctx &c) {
    if (elect_one()) tc_commit(c.bars + BAR_DRAIN * 8);
    __syncwarp();
    const unsigned long long t0 = global_ns();
    while (!mbar_try_wait(c.bars + BAR_DRAIN * 8, 0) && global_ns() - t0 < c.wait_ns + kDrainNs) {}
}

/* The row's running state after all its keys, of one query tile. */
struct RowState {
    float m, l;             /* reference (scaled log2 units) and sum */
    bool any;               /* O holds something */
    bool ok;
};

/* Where a softmax warp stands: records read, key tiles, query tiles with any. */
struct Progress {
    int r, j, done;
};

__device__ __forceinline__ RowState softmax_rows(const Ctx &c, const Params &p, const Tile &t, uint32_t tmem, const volatile Meta *meta,
                                                 Progress &at) {
    const int row = threadIdx.x & 127, lane = threadIdx.x & 31;
    const uint32_t tS = tmem + ((uint32_t)(row & ~31) << 16), tO = tS + 128;
    const bool live = (row & ~31) < t.rows;              /* this warp has rows */
    const float sl2 = p.scale_log2;
    RowState st = {-INFINITY, 0.0f, false, true};
    for (;; at.j++) {
        const int slot = at.r & (kMetaSlots - 1);
        if (!(st.ok = __all_sync(0xffffffffu, wait_bar<kFollower>(c, BAR_META + slot, (uint32_t)(at.r / kMetaSlots) & 1u, 420)))) return st;
        at.r++;
        const uint32_t state = meta[slot].state;
        auto release = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(c.bars + (BAR_META_FREE + slot) * 8);
        };
        if (is_end(state)) {
            release();
            break;
        }
        const bool begin = !st.any;
        st.any = true;
        if (!(st.ok = __all_sync(0xffffffffu, wait_bar(c, BAR_S_FULL, (uint32_t)at.j & 1u, 421)))) return st;
        tc_fence_after();
        if (!live) {
            /* Rows that do not exist: whatever lies in P only meets rows of O that nobody reads. */
            release();
            tc_fence_before();
            mbar_arrive(c.bars + BAR_P_FULL * 8);
            mbar_arrive(c.bars + (BAR_P_FULL + 1) * 8);
            continue;
        }
        uint32_t s[128];
#pragma unroll
        for (int ch = 0; ch < 4; ch++) tmem_ld32(tS + ch * 32, s + ch * 32);
        tc_wait_ld();
        if (state == kPartly) {
#pragma unroll
            for (int ch = 0; ch < 4; ch++) {
                const uint32_t bits = meta[slot].bits[ch];
                if (bits != 0xFFFFFFFFu) mask_chunk(s + ch * 32, bits);
            }
        }
        release();
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
        if (begin) {
            st.m = m_cand;
        } else {
            const bool need = m_cand > st.m + kRescaleThreshold;
            if (__any_sync(0xffffffffu, need)) {
                /* The last product is complete (it was issued before the one that filled S), the next waits for this warp. */
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
        st.ok = __all_sync(0xffffffffu, wait_bar(c, BAR_O_DONE, (uint32_t)at.done++ & 1u, 422));
        tc_fence_after();
    }
    return st;
}

/* O times f -> bf16 rows, through 4 KB of staging per warp (32 rows x 128
 * bytes, 16-byte chunks swizzled by the row): a thread owns a row, memory wants
 * eight threads per 128 bytes of it. */
__device__ __forceinline__ void store_rows(const Params &p, const Tile &t, uint32_t tmem, float f, bool any, unsigned char *stage) {
    const int row = threadIdx.x & 127, lane = threadIdx.x & 31, row0 = row & ~31;
    if (row0 >= t.rows) return;
    const uint32_t tO = tmem + ((uint32_t)row0 << 16) + 128;
    unsigned char *sw = stage + (row0 >> 5) * 4096;
    uint16_t *out = p.out + (size_t)(t.q0 + row0) * p.ldo + (size_t)t.head * kHeadDim;
#pragma unroll 1
    for (int half = 0; half < 2; half++) {
        uint32_t o[64];
        if (any) {
            tmem_ld32(tO + half * 64, o);
            tmem_ld32(tO + half * 64 + 32, o + 32);
            tc_wait_ld();
        } else {
#pragma unroll
            for (int i = 0; i < 64; i++) o[i] = 0u;
        }
#pragma unroll
        for (int ch = 0; ch < 8; ch++) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float a = __uint_as_float(o[8 * ch + 2 * e]), b = __uint_as_float(o[8 * ch + 2 * e + 1]);
                w[e] = f != 0.0f ? cvt_bf16x2(a * f, b * f) : 0u;
            }
            *reinterpret_cast<uint4 *>(sw + lane * 128 + ((ch ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int ch = lane & 7;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int r = k * 4 + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4 *>(sw + r * 128 + ((ch ^ (r & 7)) << 4));
            if (row0 + r < t.rows) *reinterpret_cast<uint4 *>(out + (size_t)r * p.ldo + half * 64 + ch * 8) = v;
        }
        __syncwarp();
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
    /* The producer sets up the barriers and starts at once; it only tells the
     * other warps, which wait here for the barriers and the tensor memory. The
     * launch is stream-serialised by program: nothing may be read or written
     * before the kernel ahead is complete, and no bounded wait may have begun.
     * (What is read may be written until then: no load through the
     * non-coherent path, which takes memory as constant for the whole kernel.) */
    uint32_t tmem = 0;
    const int shift = p.parts == 1 && blockIdx.x >= gridDim.x / 2 ? 2 : 0, producer_warp = 4 + shift, mma_warp = 5 + shift;
    if (warp == producer_warp) {
        if (lane == 0) {
            for (int b = 0; b < BAR_COUNT; b++) mbar_init(c.bars + b * 8, b == BAR_P_FULL || b == BAR_P_FULL + 1 ? 128 : b >= BAR_META_FREE ? 5 : 1);
            c.abort_flag[0] = c.abort_flag[1] = 0u;      /* and the beat */
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        asm volatile("barrier.cta.arrive.aligned 1, %0;" ::"n"(kThreads) : "memory");
    } else {
        if (warp == mma_warp) {
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
    Loads loads = {0, 0, 0};
    if (warp < 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        Progress at = {0, 0, 0};
        const int step = item_step(p);
        for (int item = first_item(p);; item += step) {
            const Tile t = tile_of(p, item, rank);
            st = softmax_rows(c, p, t, tmem, meta, at);
            if (!st.ok || p.parts > 1) break;
            store_rows(p, t, tmem, st.l != 0.0f ? 1.0f / st.l : 0.0f, st.any, smem_gen + kSmemStage);
            if (item >= p.items - step) break;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == producer_warp) loads = producer(c, p, rank, &tmq, &tmk, &tmv, smem, meta, lane);
        if (warp == mma_warp) mma_issuer(c, p, smem, smem_gen, tmem, meta, lane);
        __syncwarp();
    }

    if (p.parts > 1) {
        /* The parts of a list meet: every CTA publishes the maxima and sums of
         * its rows, scales its rows by their share of the whole and leaves them
         * in shared memory; CTA r adds the columns [r, r + 1) * 128 / parts of
         * all of them. A row that no CTA has a key for stays zero. */
        const int row = threadIdx.x & 127;
        const Tile t = tile_of(p, first_item(p), rank);
        float2 *ml = reinterpret_cast<float2 *>(smem_gen + kSmemStage);
        if (warp < 4) ml[row] = make_float2(st.m, st.l);
        cluster_sync_all();
        if (warp < 4 && (row & ~31) < t.rows) {
            float m = -INFINITY, l = 0.0f;
            for (int r = 0; r < p.parts; r++) m = fmaxf(m, ld_cluster_f2(map_to_cta(smem + kSmemStage + row * 8, r)).x);
            for (int r = 0; r < p.parts; r++) {
                const float2 o = ld_cluster_f2(map_to_cta(smem + kSmemStage + row * 8, r));
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
    /* Any warp may have given up, at any time: whether one has is known for the whole CTA only here. */
    if (warp == producer_warp) settle_loads(c, loads);
    if (warp == mma_warp) {
        if (*c.abort_flag) drain_products(c);
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
    p.unit_log = p.unit == 16 ? 4 : p.unit == 32 ? 5 : p.unit == 64 ? 6 : 7;
    p.units = kTile / p.unit;
    p.per_entry = a.k_block < kTile ? 1 : a.k_block / kTile;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.status = g.dev_status;
    p.wait_ns = wait_limit_ns();
    const long long items = (long long)a.heads * a.q_blocks * p.tiles;
    const long long key_tiles = ((long long)a.list_len * p.per_entry + p.units - 1) / p.units;
    p.per_head = a.q_blocks * p.tiles;
    p.items = (int)items;
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
    const long long slots = 2LL * g.sm_count;
    cfg.gridDim = dim3((unsigned)(p.parts > 1 ? items * p.parts : items < slots ? items : slots));
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
