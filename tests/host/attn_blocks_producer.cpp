/*
 * The producer warp of the attention over key blocks, run on host threads.
 *
 * PRODUCER_INC names a file with the kernel's own source from the first constant to the end of
 * the producer. What it calls of the device is stood in for here: a warp is 32
 * threads that meet in every collective, barriers and copies are counted. The
 * other warps of the CTA are modelled by what they wait for: the products of a
 * key tile need K, V and, once per query tile with keys, Q.
 *
 * Prints the records (key tiles with their valid keys, ends of query tiles), the
 * copies (tensor, number of the load, coordinates, place in shared memory), and
 * how many loads of Q, K and V were issued and how many of them somebody waited
 * for before the CTA may leave.
 */
#include <algorithm>
#include <atomic>
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __noinline__
#define __grid_constant__

struct CUtensorMap {
    int which;
};
struct Dim {
    unsigned x;
};
static Dim blockIdx, gridDim;

static constexpr int kLanes = 32;
static std::barrier<> g_meet(kLanes);
static int64_t g_slot[kLanes];
static thread_local int t_lane;

template <typename T> static T exchange(T mine, int src) {
    g_slot[t_lane] = (int64_t)mine;
    g_meet.arrive_and_wait();
    const T v = (T)g_slot[src & (kLanes - 1)];
    g_meet.arrive_and_wait();
    return v;
}
static uint32_t ballot(bool mine) {
    g_slot[t_lane] = mine;
    g_meet.arrive_and_wait();
    uint32_t v = 0;
    for (int i = 0; i < kLanes; i++) v |= (uint32_t)(g_slot[i] != 0) << i;
    g_meet.arrive_and_wait();
    return v;
}
static void __syncwarp() { g_meet.arrive_and_wait(); }
static int __shfl_sync(unsigned, int v, int src) { return exchange(v, src); }
static uint32_t __shfl_sync(unsigned, uint32_t v, int src) { return exchange(v, src); }
static uint32_t __ballot_sync(unsigned, bool p) { return ballot(p); }
static bool __all_sync(unsigned, bool p) { return ballot(p) == 0xFFFFFFFFu; }
static bool __any_sync(unsigned, bool p) { return ballot(p) != 0; }
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }

namespace iris_b200 {
namespace sm100 {
constexpr uint32_t idesc_bf16(int, int) { return 0; }
struct Ctx {
    uint32_t bars;
    volatile uint32_t *abort_flag;
    unsigned int *status;
    unsigned long long wait_ns;
};
static void give_up(const Ctx &c, int, unsigned) { *c.abort_flag = 1u; }
static unsigned long long global_ns() { return 0; }
/* (Defined behind the kernel's part, where its names are known.) */
static uint32_t mbar_try_wait(uint32_t bar, uint32_t parity);
static void mbar_expect_tx(uint32_t bar, uint32_t bytes);
static void mbar_arrive(uint32_t bar);
static void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar);
}  // namespace sm100
namespace attn_blocks {
using namespace sm100;
#include PRODUCER_INC
}  // namespace attn_blocks

using namespace attn_blocks;

static volatile Meta g_meta[kMetaSlots];
static int g_issued[3], g_waited[3];            /* copies of Q, K, V */
static int g_emptied[3];                        /* key tiles whose products with K, V somebody saw to their end */
static long long g_bytes[3], g_expected[3];
static bool g_with_keys;
static int g_records, g_give_up;                /* records published; how many of them the other warps live to see */
static volatile uint32_t g_abort[2];
static int g_unit;                              /* rows of a box of K or V */
struct Box {
    int which, load, x, row;
    uint32_t at;
};
static std::vector<Box> g_boxes;
static int which_of(uint32_t bar) {
    switch (bar / 8) {
        case BAR_Q_FULL: return 0;
        case BAR_K_FULL: return 1;
        case BAR_V_FULL: return 2;
    }
    fprintf(stderr, "a copy that signals barrier %u\n", bar / 8);
    exit(2);
}

namespace sm100 {
/* Everything that is waited for has happened, as long as nobody gave up; what the producer itself waits for of its copies is noted. */
static uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    if (g_abort[0] && (int)(bar / 8) != BAR_Q_FULL && (int)(bar / 8) != BAR_K_FULL && (int)(bar / 8) != BAR_V_FULL) return 0;
    if (t_lane != 0) return 1;
    const int b = (int)(bar / 8);
    /* (Arrivals of the tensor cores: one for every key tile whose products were issued.) */
    if (b == BAR_K_EMPTY || b == BAR_V_EMPTY) {
        const int w = b == BAR_K_EMPTY ? 1 : 2;
        if (((g_issued[w] - 1) & 1) == (int)parity) g_emptied[w] = g_issued[w];
    }
    if (b == BAR_Q_FULL || b == BAR_K_FULL || b == BAR_V_FULL) {
        const int w = which_of(bar);
        if (((g_issued[w] - 1) & 1) == (int)parity) g_waited[w] = std::max(g_waited[w], g_issued[w]);
    }
    return 1;
}
static void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    const int w = which_of(bar);
    g_issued[w]++;
    g_expected[w] += bytes;
}
static void mbar_arrive(uint32_t bar) {
    const int slot = (int)(bar / 8) - BAR_META;
    if (slot < 0 || slot >= kMetaSlots || slot != g_records % kMetaSlots) {
        fprintf(stderr, "record %d in slot %d\n", g_records, slot);
        exit(2);
    }
    g_records++;
    const volatile Meta &m = g_meta[slot];
    if (is_end(m.state)) {
        printf("end%s\n", m.state == kEndUnused ? " unused" : "");
        g_with_keys = false;
        return;
    }
    /* The products of the tile wait for its K and V, the first of a query tile for Q; who has given up waits for nothing. */
    if (g_records > g_give_up) g_abort[0] = 1u;
    if (!g_abort[0]) {
        if (!g_with_keys) g_waited[0] = g_issued[0];
        g_waited[1]++;
        g_waited[2]++;
    }
    g_with_keys = true;
    printf("keys %s %08x %08x %08x %08x\n", m.state == kWhole ? "whole" : "partly", m.bits[0], m.bits[1], m.bits[2], m.bits[3]);
}
static std::atomic_flag g_lock = ATOMIC_FLAG_INIT;
static void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    while (g_lock.test_and_set()) {}
    const int w = which_of(bar);
    g_bytes[w] += map->which == 0 ? kHalfBytes : g_unit * 128;
    g_boxes.push_back({map->which, g_issued[w] - 1, x, y, dst});
    g_lock.clear();
}
}  // namespace sm100
}  // namespace iris_b200

/* Arguments: seq_q seq_k heads group list_len q_block k_block rank parts part_len block grid, the record at which the others
 * give up (0: none), then the list, then seq_k mask words (or none). */
int main(int argc, char **argv) {
    using namespace iris_b200;
    using namespace iris_b200::attn_blocks;
    std::vector<int> a;
    for (int i = 1; i < argc; i++) a.push_back(atoi(argv[i]));
    if (a.size() < 13) return 2;
    Params p = {};
    p.seq_q = a[0];
    p.seq_k = a[1];
    p.heads = a[2];
    p.group = a[3];
    p.list_len = a[4];
    p.q_block = a[5];
    p.k_block = a[6];
    const int rank = a[7];
    p.parts = a[8];
    p.part_len = a[9];
    blockIdx.x = (unsigned)a[10];
    gridDim.x = (unsigned)a[11];
    p.q_blocks = (p.seq_q + p.q_block - 1) / p.q_block;
    p.k_blocks = (p.seq_k + p.k_block - 1) / p.k_block;
    p.tiles = (p.q_block + kTile - 1) / kTile;
    p.unit = p.k_block < kTile ? p.k_block : kTile;
    p.unit_log = p.unit == 16 ? 4 : p.unit == 32 ? 5 : p.unit == 64 ? 6 : 7;
    p.units = kTile / p.unit;
    g_unit = p.unit;
    p.per_entry = p.k_block < kTile ? 1 : p.k_block / kTile;
    p.per_head = p.q_blocks * p.tiles;
    p.items = p.heads * p.per_head;
    p.wait_ns = 1;
    const size_t nlist = (size_t)p.heads * p.q_blocks * p.list_len;
    if (a.size() != 13 + nlist && a.size() != 13 + nlist + (size_t)p.seq_k) return 2;
    p.list = a.data() + 13;
    p.key_mask = a.size() > 13 + nlist ? a.data() + 13 + nlist : nullptr;
    unsigned int status[8] = {};
    g_give_up = a[12] ? a[12] - 1 : 1 << 30;
    p.status = status;
    const CUtensorMap maps[3] = {{0}, {1}, {2}};
    std::vector<std::thread> warp;
    for (int lane = 0; lane < kLanes; lane++)
        warp.emplace_back([&, lane] {
            t_lane = lane;
            Ctx c = {0, g_abort, status, 1};
            const Loads n = producer(c, p, rank, &maps[0], &maps[1], &maps[2], 0, g_meta, lane);
            __syncwarp();
            settle_loads(c, n);
        });
    for (auto &t : warp) t.join();
    for (const Box &b : g_boxes)
        printf("box %c %d %d %d %u\n", "QKV"[b.which], b.load, b.x, b.row, b.at);
    for (int w = 0; w < 3; w++) {
        printf("copies %c issued %d waited %d\n", "QKV"[w], g_issued[w], g_waited[w]);
        if (w) printf("products %c issued %d waited %d\n", "QKV"[w], g_issued[w], g_emptied[w]);
        if (g_bytes[w] != g_expected[w]) return 4;
    }
    return g_abort[0] != (a[12] != 0) ? 3 : 0;
}
