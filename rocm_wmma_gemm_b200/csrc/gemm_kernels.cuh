// Device kernels of the B200 GEMM library.
//
//   gemm_umma_kernel   persistent, warp-specialised tcgen05 GEMM; one CTA per 128 x BN tile or a
//                      CTA pair per 256 x BN tile
//   splitk_reduce_kernel   deterministic sum of split-K partials + conversion to the output type
//   gemm_generic_kernel    CUDA-core GEMM for shapes whose leading dimensions TMA cannot address
//
// "Kernel view" of a problem: D (Mk x Nk, row-major) = A' (Mk x K) * B' (K x Nk) where each
// operand is either K-major (K contiguous) or MN-major (its M or N extent contiguous).  The
// host maps the reference's eight layout combinations onto this view; a column-major C is
// the row-major C^T = B^T * A^T, i.e. the operands swap roles
// (reference semantics: rocm_wmma_gemm/include/rocm_wmma_gemm/gemm.hpp:50-73).
#pragma once

#include "epilogue.cuh"
#include "ptx_sm100.cuh"

#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200 {

// ---------------------------------------------------------------------------------------------
// Launch timeline (builds with -DB200_GEMM_TIMELINE only; the macros are empty otherwise).
// CTA 0 of every GEMM launch stamps clock64() at fixed points of its three roles into one row
// of g_timeline (64 rows, used round-robin; slots 0 and 15 hold globaltimer values instead),
// and every CTA stamps globaltimer at its first load, at the end of its main loop and at its
// end into g_cta_times: where a launch spends its time between the dependency wait and the
// last store, and how evenly the CTAs of a grid finish.  Read back by b200_gemm_debug_timeline /
// b200_gemm_debug_cta_times (gemm_lib.cu) and printed by rocm_wmma_gemm_b200/timeline.py.
//   0 entry (globaltimer)  1 entry  2 set-up done  3 dependency wait done (producer)
//   4 first TMA load issued  5 last TMA load issued  6 first ring slot full (MMA thread)
//   7 last accumulator committed  8 MMAs drained  9 accumulator seen by the epilogue
//   10 first store issued  11 last store issued  12 staging buffers read  13 tail barrier
//   14 TMEM freed  15 producer ready to wait (globaltimer)
//   cluster K partitions: 16 before / 17 after the first cluster barrier  18 partials sent
//   19 after the second barrier  20 sums stored  21 staging buffers read
// ---------------------------------------------------------------------------------------------
#ifdef B200_GEMM_TIMELINE
constexpr int TIMELINE_ROWS = 64, TIMELINE_SLOTS = 24, TIMELINE_CTAS = 1024;
__device__ unsigned long long g_timeline[TIMELINE_ROWS * TIMELINE_SLOTS];
__device__ unsigned int       g_timeline_count;
__device__ unsigned long long g_cta_times[3 * TIMELINE_CTAS];
#define B200_TL(slot)                                                   \
    do {                                                                \
        if (blockIdx.x == 0) g_timeline[tl_base + (slot)] = clock64(); \
    } while (0)
#define B200_TLG(slot)                                                                 \
    do {                                                                               \
        if (blockIdx.x == 0) g_timeline[tl_base + (slot)] = ptx::global_timer_ns();   \
    } while (0)
#define B200_TL_CTA(row)                                                                                         \
    do {                                                                                                         \
        if (blockIdx.x < TIMELINE_CTAS) g_cta_times[(row) * TIMELINE_CTAS + blockIdx.x] = ptx::global_timer_ns(); \
    } while (0)
#else
#define B200_TL(slot) do { } while (0)
#define B200_TLG(slot) do { } while (0)
#define B200_TL_CTA(row) do { } while (0)
#endif

// Output element kinds of the epilogue.
enum : int { OUT_F32 = 0, OUT_F16 = 1, OUT_BF16 = 2 };

// Bits of the device status word (set when a bounded wait expires).
enum : unsigned int {
    ST_PRODUCER_WAIT = 1u,  // TMA producer waiting for a free ring slot
    ST_MMA_WAIT_FULL = 2u,  // MMA issuer waiting for a filled ring slot
    ST_MMA_WAIT_ACC  = 4u,  // MMA issuer waiting for a drained accumulator
    ST_EPI_WAIT      = 8u,  // epilogue waiting for a finished accumulator
    ST_DRAIN_WAIT    = 16u, // tail waiting for outstanding MMAs / loads
    ST_PEER_WAIT     = 32u  // CTA-pair handshake
};

struct GemmParams {
    uint32_t M, N, K;      // kernel-view extents
    uint32_t batch;        // batch count
    uint32_t m_tiles;      // ceil(M / (128 * cluster))
    uint32_t n_tiles;      // ceil(N / BN)
    uint32_t k_blocks;     // ceil(K / 64)
    uint32_t split_k;      // K partitions (>= 1); every partition owns >= 1 k-block
    uint32_t kb_per_split; // k-blocks per partition
    uint32_t group_m;      // raster band height in tiles (0 = sweep columns)
    uint32_t num_work;     // batch * split_k * m_tiles * n_tiles
    uint32_t a_mn_major;   // 0: A' K-major, 1: A' M-major
    uint32_t b_mn_major;   // 0: B' K-major, 1: B' N-major
    uint32_t idesc;        // tcgen05 instruction descriptor
    uint32_t stages;       // ring depth actually used (<= MAX_STAGES)
    unsigned int* status;  // device status word
    void*    out;          // transposed epilogue only: base of the (Nk x Mk, row-major) output
    uint32_t k_skew;       // work unit w starts its K loop (w * k_skew) k-blocks in (0 = in order)
    uint32_t stagger;      // 512-wide tiles: k-blocks by which the two column halves are staggered
    uint32_t bm;           // one-CTA kernels: rows of A' per tile (128; 8 .. 128 with the transposed epilogue)
    uint32_t wn;           // CTA-pair kernels up to 256 columns: columns per tile actually used (<= BN)
    uint32_t kc;           // one-CTA kernels: k-blocks per ring slot (1, 2 or 4)
    uint32_t k4d;          // one-CTA kernels: K-major operands use the 4-D (chunked K) maps
    uint32_t snake;        // raster: odd bands (odd columns of a column sweep) run backwards
    uint32_t l2_hints;     // L2 eviction priorities: bits [0,2) A', [2,4) B', [4,6) D (L2_HINT_*)
    uint32_t balanced;     // 1: balanced (stream-K) schedule, see WorkCursor
    uint32_t units_per_tile; // balanced: K steps (ring slots of kc k-blocks) per tile
    uint32_t workers;      // balanced: runs the cut tiles' K loops are divided into (<= persistent CTAs / CTA pairs)
    uint32_t total_units;  // balanced: sk_tiles x units_per_tile
    uint32_t sk_tiles;     // balanced: tiles [0, sk_tiles) are cut into runs; tiles [sk_tiles, num_work) are dealt whole
    uint32_t ndst;         // gathering kernels: number of destination matrices every tile is stored to
    uint32_t dst_row0;     // gathering kernels: row and column of D(0, 0) within each destination
    uint32_t dst_col0;
    uint32_t cluster_k;    // 1: the split_k K partitions of a tile are the CTAs of one cluster, summed through
                           //    distributed shared memory (work items are tiles; the cluster rank is the partition)
};

// Destinations of a gathering kernel: one tensor map per copy of the full output matrix (this
// GPU's own and its peers'), all of the same shape.
constexpr int MAX_GATHER_DST = 8;
struct GatherMaps {
    CUtensorMap m[MAX_GATHER_DST];
};

// L2 eviction priority of one operand's TMA traffic (GemmParams::l2_hints).
enum : uint32_t { L2_HINT_NONE = 0u, L2_HINT_EVICT_FIRST = 1u, L2_HINT_EVICT_LAST = 2u };

constexpr int      BLOCK_M        = 128;
constexpr int      BLOCK_K        = 64; // 64 x 2 B = one 128-byte swizzle row
constexpr int      UMMA_K         = 16;
constexpr int      MAX_STAGES     = 12; // ring depth of the staged-epilogue kernels
constexpr int      MAX_SLAB_STAGES = 24; // ring depth of the transposed-epilogue (slab) kernels
constexpr int      GEMM_THREADS   = 192; // warp 0 TMA, warp 1 MMA, warps 2..5 epilogue
constexpr int      EPI_WARPS      = 8;   // kernels with an epilogue (activation ...): warps 2..9, two per TMEM lane quarter
constexpr int      EPI_SETS       = EPI_WARPS / 4; // warps that share a lane quarter: they take its column chunks in turn
constexpr int      EPI_THREADS    = 64 + 32 * EPI_WARPS;
constexpr uint32_t A_TILE_BYTES   = BLOCK_M * BLOCK_K * 2;
constexpr uint32_t EPI_BUF_BYTES  = 32 * 128; // one warp's 32 rows x 128 B
constexpr uint32_t EPI_BYTES      = 4 * 2 * EPI_BUF_BYTES;
// Dynamic shared memory a kernel with an epilogue may use: 227 KiB minus its static part (barriers
// and two tiles' biases).
__host__ __device__ constexpr uint32_t epilogue_smem_limit(int out) { return 232448u - (out == OUT_F32 ? 2560u : 1536u); }
constexpr uint64_t WAIT_LIMIT_NS  = 2000000000ull; // 2 s per bounded wait

// Bytes of one ring slot in one CTA: A' 128 x 64 plus B' (bn / cluster) x 64.
__host__ __device__ constexpr uint32_t stage_bytes(int bn, int cluster)
{
    return A_TILE_BYTES + static_cast<uint32_t>(bn / cluster) * BLOCK_K * 2;
}

// Dynamic shared memory a launch needs (1 KiB slack for manual 1024-byte alignment).  The
// transposed epilogue stores straight from registers and needs no staging.
__host__ __device__ constexpr uint32_t gemm_smem_bytes(int bn, int cluster, int stages, bool transposed = false)
{
    return static_cast<uint32_t>(stages) * stage_bytes(bn, cluster) + (transposed ? 0u : EPI_BYTES) + 1024;
}

// Transposed-epilogue kernels stage `bm` <= 128 rows of A' per slot (a "slab"): the MMA still
// reads 128 rows, so the ring is followed by the slack the last slot's read runs into.
constexpr uint32_t SLAB_SMEM_LIMIT = 232448u - 1024u; // 227 KiB minus the static barriers
// A slot holds `kc` consecutive k-blocks of both operands (one TMA instruction per operand
// fetches all of them: the per-slot barrier and issue work is amortised over kc k-blocks).
__host__ __device__ constexpr uint32_t slab_stage_bytes(int bm, int bn, int kc)
{
    return static_cast<uint32_t>(kc) * static_cast<uint32_t>(bm + bn) * BLOCK_K * 2;
}
// The MMA reads 128 rows of A' whatever the slab height, i.e. up to 16 KiB (K-major) or kc x 8 KiB
// (a 64-row M-major slab) past the last slot: the ring is followed by that much slack.
__host__ __device__ constexpr uint32_t slab_slack_bytes(int kc)
{
    return kc * 8192u > 16384u ? kc * 8192u : 16384u;
}
__host__ __device__ constexpr uint32_t slab_smem_bytes(int bm, int bn, int kc, int stages)
{
    return static_cast<uint32_t>(stages) * slab_stage_bytes(bm, bn, kc) + slab_slack_bytes(kc) + 1024;
}
__host__ __device__ constexpr int slab_max_stages(int bm, int bn, int kc)
{
    int s = static_cast<int>((SLAB_SMEM_LIMIT - 1024u - slab_slack_bytes(kc)) / slab_stage_bytes(bm, bn, kc));
    return s > MAX_SLAB_STAGES ? MAX_SLAB_STAGES : s;
}

// One-CTA kernels with the staged epilogue and kc k-blocks per slot.
__host__ __device__ constexpr uint32_t slot_smem_bytes(int bn, int kc, int stages)
{
    return static_cast<uint32_t>(stages) * kc * stage_bytes(bn, 1) + EPI_BYTES + 1024;
}
__host__ __device__ constexpr int slot_max_stages(int bn, int kc)
{
    int s = static_cast<int>((232448u - 512u - EPI_BYTES - 1024u) / (kc * stage_bytes(bn, 1)));
    return s > MAX_STAGES ? MAX_STAGES : s;
}

// Deepest ring that fits the 227 KiB a CTA may use (static barriers included).
__host__ __device__ constexpr int max_stages(int bn, int cluster, bool transposed = false)
{
    int s = static_cast<int>((232448u - 512u - (transposed ? 0u : EPI_BYTES) - 1024u) / stage_bytes(bn, cluster));
    return s > MAX_STAGES ? MAX_STAGES : s;
}

// Waits for the phase with the given parity; gives up after WAIT_LIMIT_NS or as soon as
// another role of this CTA has given up.  Returns false on give-up.  CLUSTER_SCOPE selects an
// acquire at cluster scope (the arrivals come from the peer CTA's threads).
template <bool CLUSTER_SCOPE = false>
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity,
                                             volatile uint32_t* s_abort, unsigned int* status,
                                             unsigned int code)
{
    auto try_wait = [&]() {
        if constexpr (CLUSTER_SCOPE) return ptx::mbar_try_wait_cluster(bar, parity);
        else return ptx::mbar_try_wait(bar, parity);
    };
    // The common case is a short wait: try_wait itself blocks for a while, so the timer (a slow
    // read) and the abort flag are only looked at every 128 failed attempts, and the deadline
    // starts at the first look.
    if constexpr (!CLUSTER_SCOPE) {
        if (ptx::mbar_test_wait(bar, parity)) return true; // already complete: no blocking wait
    }
    uint64_t t0    = 0;
    uint32_t spins = 0;
    while (true) {
        if (try_wait()) return true;
        if ((++spins & 127u) == 0u) {
            if (*s_abort != 0u) return false;
            const uint64_t now = ptx::global_timer_ns();
            if (t0 == 0) {
                t0 = now;
            } else if (now - t0 > WAIT_LIMIT_NS) {
                *s_abort = 1u;
                atomicOr(status, code);
                return false;
            }
        }
    }
}

struct WorkCoord {
    uint32_t m0, n0;   // first row / column of the tile
    uint32_t z_in;     // batch index (third TMA coordinate of A' and B')
    uint32_t z_out;    // third TMA coordinate of D: batch * split_k + split
    uint32_t kb0, kb1; // k-block range
    uint32_t partial;  // balanced schedule: the segment is only part of its tile's K loop (f32 partial to the workspace)
    // kernels with an epilogue only
    uint32_t z_a, z_b; // third TMA coordinates of A' and B' (grouped products: 0, or the group)
    uint32_t k_first;  // ragged K: first row of the group (0 otherwise)
    uint32_t end;      // end of the ragged extent's group: rows (columns with the transposed epilogue) from here on are not ours
    uint32_t group, first; // group, its first row
    uint32_t wn;       // balanced ragged tiles: the tile's width
};

// Tile index -> (tile-row, tile-column) under the problem's raster.
// Raster (the reference's tile_mapper, kernel/mapping.hpp:108-287): tiles are walked in bands
// of group_m tile-rows, tile-rows fastest, so that the tiles in flight share a panel of A'
// and a few panels of B' in L2.  With `snake` every other band runs its columns backwards
// (and every other column its rows): the first tiles of a band reuse the B' panels the last
// tiles of the band before it have just read.
__device__ __forceinline__ void tile_coords(const GemmParams& p, uint32_t t, uint32_t& m_idx, uint32_t& n_idx)
{
    if (p.group_m == 0u) {
        m_idx = t % p.m_tiles;
        n_idx = t / p.m_tiles;
        if (p.snake && (n_idx & 1u)) m_idx = p.m_tiles - 1u - m_idx;
    } else {
        const uint32_t per_group = p.group_m * p.n_tiles;
        const uint32_t g         = t / per_group;
        const uint32_t first_m   = g * p.group_m;
        const uint32_t gsize     = min(p.group_m, p.m_tiles - first_m);
        const uint32_t in_g      = t - g * per_group;
        uint32_t       m_in      = in_g % gsize;
        n_idx                    = in_g / gsize;
        if (p.snake) {
            if (n_idx & 1u) m_in = gsize - 1u - m_in;
            if (g & 1u) n_idx = p.n_tiles - 1u - n_idx;
        }
        m_idx = first_m + m_in;
    }
}

__device__ __forceinline__ WorkCoord decode_work(const GemmParams& p, uint32_t w, int bn, int bm, uint32_t krank)
{
    const uint32_t tiles = p.m_tiles * p.n_tiles;
    const uint32_t t     = w % tiles;
    const uint32_t r     = w / tiles;
    const uint32_t split = p.cluster_k ? krank : r % p.split_k;
    const uint32_t b     = p.cluster_k ? r : r / p.split_k;
    uint32_t       m_idx, n_idx;
    tile_coords(p, t, m_idx, n_idx);
    WorkCoord c;
    c.m0    = m_idx * static_cast<uint32_t>(bm);
    c.n0    = n_idx * static_cast<uint32_t>(bn);
    c.z_in  = b;
    c.z_out = p.cluster_k ? b : b * p.split_k + split;
    c.kb0   = split * p.kb_per_split;
    c.kb1   = min(p.k_blocks, c.kb0 + p.kb_per_split);
    c.partial = 0u;
    return c;
}

// ---------------------------------------------------------------------------------------------
// Work of one persistent worker (a CTA, or a CTA pair).
//
// Plain schedule: work items unit, unit + units, ... of the num_work (batch x K partition x
// tile) items.
//
// Balanced schedule (stream-K; the reference's roadmap names it, README.md:202).  Whole waves
// of tiles need no balancing, so only the tiles of the incomplete wave - sk_tiles = tiles mod
// workers, or all of them when there are fewer tiles than workers - are cut: their K loops are
// laid end to end - tile 0's K steps, then tile 1's, ... - and that line of total_units steps
// is cut into `workers` equal runs, one per worker, wherever the cuts fall.  A worker first
// walks its run segment by segment (a segment = the part of one tile's K loop inside the run)
// and then takes whole tiles sk_tiles + worker, sk_tiles + worker + grid, ... like the plain
// schedule: every SM gets the same number of K steps whatever the tile count, and the cut
// tiles' partials are written early in the kernel, not at its end.  A segment that covers a
// tile's whole K loop stores the tile to C like the plain schedule does.  A partial segment
// leaves an f32 partial tile in the workspace: a run has at most two of them, its first (it
// starts inside a tile: slot 2 * worker) and its last (it ends inside a tile: slot
// 2 * worker + 1); the fix-up pass (streamk_reduce_kernel) adds a split tile's partials in
// K order and writes C.  No CTA waits for another.
// ---------------------------------------------------------------------------------------------
struct WorkCursor {
    uint32_t next;  // plain: next work item; balanced: next K step of the run
    uint32_t end;   // balanced: end of the run
    uint32_t krank; // cluster K partitions: this CTA's partition (its rank in the cluster)
    uint32_t dp;    // balanced: next whole tile of this worker
};

__device__ __forceinline__ uint32_t run_start(const GemmParams& p, uint32_t worker)
{
    return static_cast<uint32_t>(static_cast<uint64_t>(worker) * p.total_units / p.workers);
}

__device__ __forceinline__ WorkCursor work_begin(const GemmParams& p, uint32_t unit, uint32_t krank = 0u)
{
    WorkCursor cur;
    cur.krank = krank;
    cur.dp = 0u;
    if (p.balanced) {
        const bool has_run = unit < p.workers;
        cur.next = has_run ? run_start(p, unit) : 0u;
        cur.end  = has_run ? run_start(p, unit + 1u) : 0u;
        cur.dp   = p.sk_tiles + unit;
    } else {
        cur.next = unit;
        cur.end  = p.num_work;
    }
    return cur;
}

// Next piece of work of this worker; false when there is none left.
__device__ __forceinline__ bool work_next(const GemmParams& p, WorkCursor& cur, uint32_t unit, uint32_t units,
                                          int bn, int bm, WorkCoord& c)
{
    if (!p.balanced) {
        if (cur.next >= cur.end) return false;
        c = decode_work(p, cur.next, bn, bm, cur.krank);
        cur.next += units;
        return true;
    }
    if (cur.next >= cur.end) { // the run is done: whole tiles, round-robin over the grid
        if (cur.dp >= p.num_work) return false;
        const uint32_t tiles = p.m_tiles * p.n_tiles;
        uint32_t       m_idx, n_idx;
        tile_coords(p, cur.dp % tiles, m_idx, n_idx);
        c.m0      = m_idx * static_cast<uint32_t>(bm);
        c.n0      = n_idx * static_cast<uint32_t>(bn);
        c.z_in    = cur.dp / tiles;
        c.z_out   = c.z_in;
        c.partial = 0u;
        c.kb0     = 0u;
        c.kb1     = p.k_blocks;
        cur.dp += units;
        return true;
    }
    const uint32_t tile  = cur.next / p.units_per_tile;          // over batch x tiles
    const uint32_t first = cur.next - tile * p.units_per_tile;   // first K step of the segment within the tile
    const uint32_t last  = min(p.units_per_tile, first + (cur.end - cur.next));
    const uint32_t tiles = p.m_tiles * p.n_tiles;
    uint32_t       m_idx, n_idx;
    tile_coords(p, tile % tiles, m_idx, n_idx);
    c.m0    = m_idx * static_cast<uint32_t>(bm);
    c.n0    = n_idx * static_cast<uint32_t>(bn);
    c.z_in    = tile / tiles;
    c.partial = (first != 0u || last != p.units_per_tile) ? 1u : 0u;
    // whole tile: third coordinate of C (the batch index); partial: the workspace slot
    c.z_out   = c.partial ? 2u * unit + (first != 0u ? 0u : 1u) : c.z_in;
    c.kb0     = first * p.kc;
    c.kb1     = min(p.k_blocks, last * p.kc);
    cur.next += last - first;
    return true;
}

// ---------------------------------------------------------------------------------------------
// Work of the kernels with an epilogue.  Dense problems: the plain schedule.  Ragged rows: the
// groups' tiles one group after the other, within a group the ragged extent fastest, so that the
// tiles in flight share the group's matrix; ragged K: every group has the same tiles, its K loop
// runs over its own rows.  The group table (sanitised first rows, running tile counts) is built
// in shared memory by build_group_table.
// ---------------------------------------------------------------------------------------------
struct GroupTable {
    const uint32_t* first; // groups + 1 row offsets
    const uint32_t* tiles; // groups + 1 running counts of ragged tiles (ragged rows only)
};

// By one warp.
__device__ __forceinline__ void build_group_table(const EpilogueParams& ep, uint32_t tile, uint32_t* first, uint32_t* tiles)
{
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t       before = 0u;
    if (lane == 0) tiles[0] = 0u;
    for_each_group(ep.offsets, ep.groups, ep.rows, [&](uint32_t g, uint32_t lo, uint32_t hi) {
        const uint32_t incl = before + warp_scan_add((hi - lo + tile - 1u) / tile, lane);
        if (g < ep.groups) {
            first[g]      = lo;
            tiles[g + 1u] = incl;
            if (g + 1u == ep.groups) first[ep.groups] = hi;
        }
        before = __shfl_sync(0xffffffffu, incl, 31);
        return false;
    });
}

// tile_coords with the divisors the host has prepared.
__device__ __forceinline__ void tile_coords_epilogue(const GemmParams& p, const EpilogueParams& ep, uint32_t t, uint32_t& m_idx, uint32_t& n_idx)
{
    if (p.group_m == 0u) {
        n_idx = fast_div(t, ep.per_column);
        m_idx = t - n_idx * p.m_tiles;
        if (p.snake && (n_idx & 1u)) m_idx = p.m_tiles - 1u - m_idx;
        return;
    }
    const uint32_t g       = fast_div(t, ep.per_band);
    const uint32_t first_m = g * p.group_m;
    const uint32_t gsize   = min(p.group_m, p.m_tiles - first_m);
    const uint32_t in_g    = t - g * p.group_m * p.n_tiles;
    n_idx                  = gsize == ep.per_column.d ? fast_div(in_g, ep.per_column) : in_g / gsize; // (the last band may be lower)
    uint32_t m_in          = in_g - n_idx * gsize;
    if (p.snake) {
        if (n_idx & 1u) m_in = gsize - 1u - m_in;
        if (g & 1u) n_idx = p.n_tiles - 1u - n_idx;
    }
    m_idx = first_m + m_in;
}

//
// BALANCED (ragged rows along N, see the pair kernel with the transposing epilogue): a group's tiles are
// equally wide, multiples of 32 columns, instead of bn wide with a narrow last one.
template <bool TR, bool BALANCED = false>
__device__ __forceinline__ bool work_next_epilogue(const GemmParams& p, const EpilogueParams& ep, const GroupTable& gt,
                                                   WorkCursor& cur, uint32_t units, int bn, int bm, WorkCoord& c)
{
    const uint32_t w = cur.next;
    cur.next += units;
    c.partial = 0u;
    if (ep.ragged != RAGGED_ROWS) { // dense (the K partitions of a tile are one cluster's CTAs), or ragged K
        if (w >= p.num_work) return false;
        const uint32_t b = fast_div(w, ep.per_item);
        uint32_t       m_idx, n_idx;
        tile_coords_epilogue(p, ep, w - b * ep.per_item.d, m_idx, n_idx);
        c.m0   = m_idx * static_cast<uint32_t>(bm);
        c.n0   = n_idx * static_cast<uint32_t>(bn);
        c.z_in = c.z_out = b;
        c.end  = TR ? p.N : p.M;
        if (ep.ragged == RAGGED_K) {
            c.group = b;
            c.first = c.k_first = gt.first[b];
            c.z_a = c.z_b = c.kb0 = 0u;
            c.kb1 = (gt.first[b + 1u] - c.first + BLOCK_K - 1u) / BLOCK_K;
        } else {
            c.z_a = c.z_b = b;
            c.k_first = c.group = c.first = 0u;
            c.kb0 = cur.krank * p.kb_per_split;
            c.kb1 = min(p.k_blocks, c.kb0 + p.kb_per_split);
        }
        return true;
    }
    const uint32_t other = ep.per_item.d; // tiles of the other extent
    const uint32_t wt    = fast_div(w, ep.per_item);
    if (wt >= gt.tiles[ep.groups]) return false;
    uint32_t lo = 0u, hi = ep.groups; // the group whose tiles [tiles[e], tiles[e + 1]) hold wt
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (gt.tiles[mid] <= wt) lo = mid;
        else hi = mid;
    }
    const uint32_t t0    = gt.tiles[lo];
    const uint32_t in_g  = w - t0 * other;
    const uint32_t rt    = gt.tiles[lo + 1u] - t0;
    const uint32_t o     = rt == 1u ? in_g : in_g / rt;
    c.group              = lo;
    c.first              = gt.first[lo];
    c.end                = gt.first[lo + 1u];
    // (rt tiles of at most bn columns: the last one begins before the group ends whatever their width)
    c.wn                 = BALANCED ? ((c.end - c.first + rt - 1u) / rt + 31u) & ~31u : static_cast<uint32_t>(TR ? bn : bm);
    const uint32_t along = c.first + (in_g - o * rt) * c.wn;
    c.m0                 = TR ? o * static_cast<uint32_t>(bm) : along;
    c.n0                 = TR ? along : o * static_cast<uint32_t>(bn);
    c.z_a                = TR ? lo : 0u;
    c.z_b                = TR ? 0u : lo;
    c.z_in = c.z_out = c.k_first = c.kb0 = 0u;
    c.kb1            = p.k_blocks;
    return true;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
                 "r"(d)
                 : "memory");
}

// TMA load whose completion bytes go to `bar`: this CTA's barrier (CL = 1) or a
// shared::cluster address naming the pair leader's barrier (CL = 2).
template <int CL>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, uint32_t bar,
                                         int32_t c0, int32_t c1, int32_t c2, uint64_t policy)
{
    if constexpr (CL == 2) ptx::tma_load_3d_pair(dst, tm, bar, c0, c1, c2, policy);
    else ptx::tma_load_3d(dst, tm, bar, c0, c1, c2, policy);
}

// tcgen05.commit arriving on `bar` of this CTA (CL = 1) or of both CTAs of the pair (CL = 2).
template <int CL>
__device__ __forceinline__ void umma_arrive(uint32_t bar)
{
    if constexpr (CL == 2) ptx::umma_commit_pair(bar, 0x3);
    else ptx::umma_commit(bar);
}

// Schedule of a 512-wide tile (two 256-column halves that share the staged A' tile).
// With a stagger of X k-blocks a work unit of nkb k-blocks runs nkb + X steps:
//   steps [0, X)          half 0 alone on k-blocks 0 .. X-1
//   steps [X, nkb)        both halves on k-block s (one A' tile feeds two MMAs)
//   steps [nkb, nkb + X)  half 1 alone on k-blocks 0 .. X-1 (its K order is rotated by X)
// Half 0 is complete X steps before half 1, so its accumulator drains while half 1 finishes,
// and half 1 drains under the next tile's half-0-only steps: the tensor pipe does not wait for
// the epilogue although one tile fills all 512 TMEM columns.  Cost: A' k-blocks 0 .. X-1 are
// staged twice.
struct TileStep {
    uint32_t kb_rel; // k-block relative to the work unit's first
    uint32_t mask;   // bit h set: column half h takes part
};

__device__ __forceinline__ TileStep tile_step(uint32_t s, uint32_t nkb, uint32_t stagger)
{
    TileStep t;
    if (s < stagger) {
        t.kb_rel = s;
        t.mask   = 1u;
    } else if (s < nkb) {
        t.kb_rel = s;
        t.mask   = 3u;
    } else {
        t.kb_rel = s - nkb;
        t.mask   = 2u;
    }
    return t;
}

template <int OUT>
__device__ __forceinline__ uint32_t pack2(uint32_t lo_bits, uint32_t hi_bits)
{
    const float lo = __uint_as_float(lo_bits);
    const float hi = __uint_as_float(hi_bits);
    if constexpr (OUT == OUT_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// ---------------------------------------------------------------------------------------------
// Persistent tcgen05 GEMM.  CL = 1: one CTA per 128 x BN output tile.  CL = 2: a cluster of two
// CTAs (a "pair", ranks 0 and 1) per 256 x BN tile; each CTA loads its own 128 rows of A' and
// its own BN/2 columns of B', rank 0 issues one cta_group::2 MMA per K = 16 slice that reads
// both CTAs' shared memory and writes both CTAs' TMEM (each holds its 128 rows x BN columns).
// The pair halves the B' bytes each SM has to stage per FLOP.
//
//   warp 0 (one elected lane)  TMA producer: fills a `stages`-deep ring of slots (128-byte
//                      swizzle): {A' 128x64, B' (BN/CL)x64} per slot, or - one-CTA kernels up to
//                      256 columns - kc k-blocks of {A' bm x 64, B' BN x 64}, one TMA instruction
//                      per operand.  Slot s has a `full` barrier (bytes landed; for a pair it
//                      lives in rank 0 and counts both CTAs' bytes) and an `empty` barrier
//                      (MMAs that read the slot have retired).
//   warp 1 (one elected lane)  MMA issuer (rank 0 only for a pair): 4 x tcgen05.mma per
//                      k-block into one of the TMEM accumulators (BN f32 columns each);
//                      tcgen05.commit releases the slot and, after the last k-block, publishes
//                      the accumulator.  (The two single threads are chosen with elect.sync:
//                      the compiler then issues TMA / MMA / commit from uniform registers.)
//   warps 2..5         epilogue: tcgen05.ld 32 lanes x 32 columns, convert, swizzled store to a
//                      per-warp staging buffer, TMA store of 32 rows x 128 B; the accumulator
//                      is handed back as soon as its last column chunk is in registers, so the
//                      epilogue of tile i overlaps the main loop of tile i + 1.  TR = true:
//                      the transposing epilogue of skinny problems (direct coalesced stores).
//
// Edges: TMA zero-fills out-of-range loads (M, N and K tails) and clips stores.
// No TMA load here uses cluster multicast.
//
// EP: a product with an epilogue, dense or grouped (epilogue.cuh has the mathematics).  Eight
// epilogue warps, two per lane quarter, take the column chunks of a tile alternately: an
// activation costs 15 to 40 instructions per element, and four warps alone would pace short K
// loops.  The matrix an epilogue reads (residual, or Z in gradient mode) comes by TMA into the
// staging buffer its chunk will leave from, requested before the accumulator is awaited, so its
// latency hides under the main loop; Z leaves through a staging buffer of its own.
//
// EP && TR && CL == 2 (TRP): grouped products with more than a few rows per group.  The groups' matrices are
// A' (256 of C's columns per tile and pair), C's rows are the MMA's N, which comes in steps of 32: a
// group's rows are rounded up to 32 per tile, not to 256 as they would be along M (512 rows per
// group on average: 25 % more products than asked for).  A group's tiles are equally wide; the MMA's N
// extent is set per tile, and the box of rows is always 128 per CTA (boxes of just the rows wanted cost
// more producer instructions than they save traffic: 16384 rows in 32 groups x 2048 x 4096 272 us in
// boxes of 32, 256 in boxes of 64, 251 whole; 278 with the rows along M).
// ---------------------------------------------------------------------------------------------
// Maps of the matrices beside C: the one the epilogue reads, and where Z goes.
struct EpilogueMaps {
    CUtensorMap in, aux;
};

// The epilogues work in pieces of 16 columns, in loops that are not unrolled: the whole of a piece - bias, activation, residual, conversion - is a few
// hundred instructions, which stay in the instruction cache.
constexpr int PIECE = 16;

// Sum of v[j] over the 32 lanes: lane l receives the sum of v[l % PIECE].
__device__ __forceinline__ float warp_column_sums(float (&v)[PIECE], uint32_t lane)
{
#pragma unroll
    for (int s = PIECE / 2; s > 0; s /= 2) {
        const bool up = (lane & s) != 0u;
#pragma unroll
        for (int i = 0; i < s; ++i) {
            const float send = up ? v[i] : v[i + s];
            const float keep = up ? v[i + s] : v[i];
            v[i]             = keep + __shfl_xor_sync(0xffffffffu, send, s);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], PIECE);
}

// Accumulator columns from TMEM.  The load and its wait stay together: a load in flight across a
// branch or a loop's back edge would let the compiler copy its destination registers, and reuse
// them, before the hardware has written them.
struct TmemPieces {
    uint32_t addr;  // first column of the chunk
    uint32_t count; // pieces
    bool     empty; // nothing was accumulated: zeros

    // Piece i (in order); `done` is called once the chunk's last piece has been read.
    template <class F>
    __device__ __forceinline__ void get(uint32_t i, float (&v)[PIECE], F&& done)
    {
        if (empty) {
#pragma unroll
            for (int j = 0; j < PIECE; ++j) v[j] = 0.f;
        } else {
            uint32_t t[PIECE];
            ptx::tmem_ld_32x16(addr + i * PIECE, t);
            ptx::tmem_ld_wait(t);
#pragma unroll
            for (int j = 0; j < PIECE; ++j) v[j] = __uint_as_float(t[j]);
        }
        if (i + 1u == count) done();
    }
};

// Sums of a cluster's K partitions: this CTA's own part from TMEM, the others' from shared memory
// (laid out [16-byte unit][lane], see the cluster exchange), added in partition order.
struct ClusterPieces {
    uint32_t addr;       // this CTA's accumulator columns of the chunk
    uint32_t ring;       // partial of partition 0 of this chunk, this warp's rows, this lane
    uint32_t slot_bytes; // from one partition's to the next
    uint32_t parts, rank;

    template <class F>
    __device__ __forceinline__ void get(uint32_t i, float (&v)[PIECE], F&&) const
    {
        uint32_t own[PIECE];
        ptx::tmem_ld_32x16(addr + i * PIECE, own);
        ptx::tmem_ld_wait(own);
#pragma unroll
        for (int j = 0; j < PIECE; ++j) v[j] = 0.f;
#pragma unroll 1
        for (uint32_t s = 0; s < parts; ++s) {
            if (s == rank) {
#pragma unroll
                for (int j = 0; j < PIECE; ++j) v[j] += __uint_as_float(own[j]);
            } else {
#pragma unroll
                for (uint32_t u = 0; u < PIECE / 4; ++u) {
                    uint32_t x[4];
                    ptx::ld_shared_v4(ring + s * slot_bytes + (i * (PIECE / 4) + u) * 512u, x[0], x[1], x[2], x[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * u + k] += __uint_as_float(x[k]);
                }
            }
        }
    }
};

// Element-wise steps of an epilogue over N values.
template <int N>
__device__ __forceinline__ void apply_activation(const EpilogueParams& ep, float (&v)[N])
{
    with_act(ep.act, [&](auto tag) {
        constexpr uint32_t ACT = decltype(tag)::value;
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 y = act_value<ACT>(make_float2(v[j], v[j + 1]), ep);
            v[j] = y.x, v[j + 1] = y.y;
        }
    });
}

template <int N>
__device__ __forceinline__ void apply_slope(const EpilogueParams& ep, float (&v)[N], const float (&z)[N])
{
    with_act(ep.act, [&](auto tag) {
        constexpr uint32_t ACT = decltype(tag)::value;
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 y = __fmul2_rn(make_float2(v[j], v[j + 1]), act_slope<ACT>(make_float2(z[j], z[j + 1]), ep));
            v[j] = y.x, v[j + 1] = y.y;
        }
    });
}

template <int N>
__device__ __forceinline__ void add_values(float* v, const float (&t)[N])
{
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float2 y = __fadd2_rn(make_float2(v[j], v[j + 1]), make_float2(t[j], t[j + 1]));
        v[j] = y.x, v[j + 1] = y.y;
    }
}

template <int OUT>
using OutType = std::conditional_t<OUT == OUT_F32, float, std::conditional_t<OUT == OUT_F16, __half, __nv_bfloat16>>;

// 16 bytes of an output type as f32 values and back.
template <int OUT>
__device__ __forceinline__ void unpack16(const uint32_t (&w)[4], float* v)
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (OUT == OUT_F32) {
            v[k] = __uint_as_float(w[k]);
        } else if constexpr (OUT == OUT_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            v[2 * k] = f.x, v[2 * k + 1] = f.y;
        } else {
            v[2 * k] = __uint_as_float(w[k] << 16), v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}

// apply_slope for Z as it is stored: N values in 16-byte units.
template <int OUT, int N, int UNITS>
__device__ __forceinline__ void apply_slope(const EpilogueParams& ep, float (&v)[N], uint32_t (&w)[UNITS][4])
{
    with_act(ep.act, [&](auto tag) {
        constexpr uint32_t ACT = decltype(tag)::value;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            constexpr int UNIT = N / UNITS;
            float         z[UNIT];
            limit_words<ACT, OutType<OUT>>(w[i]);
            unpack16<OUT>(w[i], z);
#pragma unroll
            for (int j = 0; j < UNIT; j += 2) {
                const float2 y = __fmul2_rn(make_float2(v[i * UNIT + j], v[i * UNIT + j + 1]), act_slope<ACT, OUT != OUT_F32>(make_float2(z[j], z[j + 1]), ep));
                v[i * UNIT + j] = y.x, v[i * UNIT + j + 1] = y.y;
            }
        }
    });
}

template <int OUT>
__device__ __forceinline__ void pack16(const float* v, uint32_t (&w)[4])
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (OUT == OUT_F32) w[k] = __float_as_uint(v[k]);
        else w[k] = pack2<OUT>(__float_as_uint(v[2 * k]), __float_as_uint(v[2 * k + 1]));
    }
}

// (Operands that may be absent - bias, the read matrix, offsets - are read with ordinary loads.  A
// load through the read-only path counts as safe to execute early: with no bias, the compiler moved
// `__ldg(bias + i)` out of a loop and above the test of the pointer.)

template <class T>
__device__ __forceinline__ T ld_shared_elem(uint32_t addr)
{
    if constexpr (sizeof(T) == 4) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
        return v;
    } else {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
        T t;
        *reinterpret_cast<uint16_t*>(&t) = v;
        return t;
    }
}
template <class T>
__device__ __forceinline__ void st_shared_elem(uint32_t addr, T t)
{
    if constexpr (sizeof(T) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(t) : "memory");
    else asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(*reinterpret_cast<const uint16_t*>(&t)) : "memory");
}

// One epilogue warp of a staged kernel with an epilogue: 32 rows x 128-byte column chunks.
template <int OUT>
struct EpilogueWarp {
    using T = OutType<OUT>;
    static constexpr int      CH    = OUT == OUT_F32 ? 32 : 64; // columns per chunk
    static constexpr int      PARTS = CH / 32;
    static constexpr uint32_t UNIT  = CH / 8;                   // columns per 16 bytes

    const GemmParams&        p;
    const EpilogueParams&    ep;
    const EpilogueMaps&      em;
    const CUtensorMap&       tmD;
    void*                    out;     // C, for what TMA may not store
    uint32_t                 lane;
    uint32_t                 stg;     // staging buffers: ep.bufs for C, then one for Z
    uint32_t                 in_bar;  // barriers of the first two
    uint8_t*                 bias_sm; // the tile's biases, in C's type
    volatile uint32_t*       s_abort;
    uint32_t                 count     = 0; // chunks so far: the next one's buffer is count % ep.bufs
    uint32_t                 in_phase  = 0; // parity per buffer
    uint32_t                 in_flight = 0; // requested, not yet awaited

    __device__ __forceinline__ uint32_t slot(uint32_t k) const { return (count + k) & (ep.bufs - 1u); }

    // Requests the read matrix's chunk k chunks ahead.  Its buffer must have been read by the
    // stores before (request() is called after a wait on them).
    __device__ __forceinline__ void request(uint32_t k, uint32_t row0, uint32_t col0, uint32_t z)
    {
        if (ep.unaligned) return; // (read in finish)
        const uint32_t b = slot(k);
        if (lane == 0) {
            ptx::mbar_expect_tx(in_bar + 8u * b, EPI_BUF_BYTES);
            ptx::tma_load_3d(stg + b * EPI_BUF_BYTES, &em.in, in_bar + 8u * b, col0, row0, z, 0);
        }
        in_flight |= 1u << b;
    }

    // Every store so far has read its staging buffer, and this warp's own accesses to them are done.
    __device__ __forceinline__ void buffers_free()
    {
        ptx::fence_proxy_async_smem();
        if (lane == 0) ptx::tma_store_wait_read<0>();
        __syncwarp();
    }

    // Columns [32 w, 32 w + 32) of the tile's (tile half's) biases by epilogue warp w; the barrier before
    // the accumulator orders them before their use.
    __device__ __forceinline__ void fetch_bias(const WorkCoord& c, uint32_t col0, uint32_t at, uint8_t* to)
    {
        bias_sm = to;
        if (!ep.bias || ep.bias_on_rows) return;
        const T* b = static_cast<const T*>(ep.bias) + (ep.ragged == RAGGED_ROWS ? c.group : c.z_in) * ep.bias_stride;
        reinterpret_cast<T*>(to)[at + lane] = col0 + at + lane < p.N ? b[col0 + at + lane] : from_f32<T>(0.f);
    }

    __device__ __forceinline__ float row_bias(const WorkCoord& c, uint32_t row) const
    {
        if (!ep.bias || !ep.bias_on_rows || row >= p.M) return 0.f;
        return to_f32(static_cast<const T*>(ep.bias)[c.z_in * ep.bias_stride + row]);
    }

    // Rows [row0, end) of a chunk between a staging buffer and a matrix that TMA cannot address, or a
    // block whose last rows belong to the next group: element by element, a row's 32 or 64 elements
    // at a time.
    template <bool LOAD>
    __device__ __forceinline__ void move_rows(uint32_t buf, void* base, uint32_t z, uint32_t row0, uint32_t col0, uint32_t end) const
    {
        const uint32_t rows = min(32u, end - row0);
        T*             at   = static_cast<T*>(base) + (static_cast<uint64_t>(z) * p.M + row0) * p.N + col0 + lane;
#pragma unroll 4
        for (uint32_t r = 0; r < rows; ++r, at += p.N) {
#pragma unroll
            for (uint32_t h = 0; h < static_cast<uint32_t>(PARTS); ++h) {
                const uint32_t col  = h * 32u + lane;
                const uint32_t addr = buf + r * 128u + (((col / UNIT) ^ (r & 7u)) << 4) + (col % UNIT) * static_cast<uint32_t>(sizeof(T));
                if (col0 + col < p.N) {
                    if constexpr (LOAD) st_shared_elem(addr, at[h * 32u]);
                    else at[h * 32u] = ld_shared_elem<T>(addr);
                }
            }
        }
    }

    // The staged chunk in buffer `sbuf` (and Z in `xbuf`) to memory.
    __device__ __forceinline__ void store(const WorkCoord& c, uint32_t row0, uint32_t col0, uint32_t end, uint32_t sbuf, uint32_t xbuf)
    {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (ep.unaligned || (ep.ragged == RAGGED_ROWS && row0 + 32u > end)) {
            move_rows<false>(sbuf, out, c.z_out, row0, col0, end);
            if (ep.aux) move_rows<false>(xbuf, ep.preact, c.z_out, row0, col0, end);
        } else if (lane == 0) {
            ptx::tma_store_3d(&tmD, sbuf, col0, row0, c.z_out, 0);
            if (ep.aux) ptx::tma_store_3d(&em.aux, xbuf, col0, row0, c.z_out, 0);
        }
        if (lane == 0) ptx::tma_store_commit(); // (an empty group keeps the count of the waits)
        ++count;
    }

    // The same for a chunk that is only converted: no branch but the ones above.
    template <class F>
    __device__ __forceinline__ void finish_plain(const WorkCoord& c, uint32_t row0, uint32_t col0, uint32_t end, uint32_t acc, bool empty,
                                                 F&& accumulators_read)
    {
        const uint32_t sbuf = stg + slot(0) * EPI_BUF_BYTES, row = sbuf + lane * 128u + ((lane & 7u) << 4);
        uint32_t       t[PARTS][32];
        if (empty) {
#pragma unroll
            for (int h = 0; h < PARTS; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j) t[h][j] = 0u;
        } else {
#pragma unroll
            for (int h = 0; h < PARTS; ++h) ptx::tmem_ld_32x32(acc + h * 32u, t[h]);
#pragma unroll
            for (int h = 0; h < PARTS; ++h) ptx::tmem_ld_wait(t[h]);
        }
        accumulators_read();
        if (lane == 0) {
            if (ep.bufs == 1u) ptx::tma_store_wait_read<0>();
            else ptx::tma_store_wait_read<1>();
        }
        __syncwarp();
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) {
            if constexpr (OUT == OUT_F32) {
                st_shared_v4(row ^ (u << 4), t[0][4 * u], t[0][4 * u + 1], t[0][4 * u + 2], t[0][4 * u + 3]);
            } else {
                const uint32_t* v = &t[u / 4][(u % 4) * 8];
                st_shared_v4(row ^ (u << 4), pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]), pack2<OUT>(v[4], v[5]), pack2<OUT>(v[6], v[7]));
            }
        }
        store(c, row0, col0, end, sbuf, sbuf);
    }

    // The chunk at (row0, col0), column tile_col of its tile, from its accumulators; `end` bounds the
    // rows.  False: a wait ran out.
    template <class Pieces, class F>
    __device__ __forceinline__ bool finish(const WorkCoord& c, uint32_t row0, uint32_t col0, uint32_t tile_col, uint32_t end, float bias_row,
                                           Pieces& pieces, F&& accumulators_read)
    {
        const uint32_t b    = slot(0);
        const uint32_t sbuf = stg + b * EPI_BUF_BYTES, xbuf = stg + ep.bufs * EPI_BUF_BYTES;
        // 16-byte unit u of this lane's row lies at (buffer + row_at) ^ (u << 4): the 128-byte swizzle
        const uint32_t row_at  = lane * 128u + ((lane & 7u) << 4);
        const uint32_t rowaddr = sbuf + row_at, xrow = xbuf + row_at;
        const uint32_t row  = row0 + lane;
        const bool     col_bias = ep.bias && !ep.bias_on_rows;
        const uint32_t bias_at  = ptx::smem_u32(bias_sm) + tile_col * static_cast<uint32_t>(sizeof(T));
        if (ep.streamed && ep.unaligned) {
            __syncwarp();
            move_rows<true>(sbuf, ep.gradient ? ep.preact : const_cast<void*>(ep.residual), c.z_out, row0, col0, end);
        } else if (ep.streamed) {
            bool ok = bounded_wait(in_bar + 8u * b, (in_phase >> b) & 1u, s_abort, p.status, ST_EPI_WAIT);
            ok      = __all_sync(0xffffffffu, ok);
            if (!ok) return false;
            in_phase ^= 1u << b;
            in_flight &= ~(1u << b);
        }
        // the buffers written below must have been read by the stores that last used them
        if (lane == 0) {
            if (ep.aux || ep.bufs == 1u) ptx::tma_store_wait_read<0>();
            else if (!ep.streamed) ptx::tma_store_wait_read<1>();
        }
        __syncwarp();
        float row_sum = 0.f;
#pragma unroll 1
        for (uint32_t pc = 0; pc < CH / PIECE; ++pc) {
            constexpr uint32_t UNITS = PIECE / UNIT; // 16-byte units of a row's piece
            const uint32_t first = (pc * UNITS) << 4, srow = rowaddr ^ first, xr = xrow ^ first;
            float v[PIECE];
            pieces.get(pc, v, accumulators_read);
            if (ep.gradient) {
                if (ep.streamed) {
                    uint32_t w[UNITS][4];
#pragma unroll
                    for (uint32_t i = 0; i < UNITS; ++i) ptx::ld_shared_v4(srow ^ (i << 4), w[i][0], w[i][1], w[i][2], w[i][3]);
                    apply_slope<OUT>(ep, v, w);
                }
            } else {
                if (col_bias) {
#pragma unroll
                    for (uint32_t i = 0; i < UNITS; ++i) {
                        uint32_t w[4];
                        float    t[UNIT];
                        ptx::ld_shared_v4(bias_at + (pc * UNITS + i) * 16u, w[0], w[1], w[2], w[3]);
                        unpack16<OUT>(w, t);
                        add_values(v + i * UNIT, t);
                    }
                } else if (ep.bias) {
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) v[j] += bias_row;
                }
                if (ep.aux) {
#pragma unroll
                    for (uint32_t i = 0; i < UNITS; ++i) {
                        uint32_t w[4];
                        pack16<OUT>(v + i * UNIT, w);
                        st_shared_v4(xr ^ (i << 4), w[0], w[1], w[2], w[3]);
                    }
                }
                apply_activation(ep, v);
                if (ep.streamed) {
#pragma unroll
                    for (uint32_t i = 0; i < UNITS; ++i) {
                        uint32_t w[4];
                        float    r[UNIT];
                        ptx::ld_shared_v4(srow ^ (i << 4), w[0], w[1], w[2], w[3]);
                        unpack16<OUT>(w, r);
                        add_values(v + i * UNIT, r);
                    }
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < UNITS; ++i) {
                uint32_t w[4];
                pack16<OUT>(v + i * UNIT, w);
                st_shared_v4(srow ^ (i << 4), w[0], w[1], w[2], w[3]);
            }
            if (ep.part) {
                // (what lies outside C may be NaN: a zero-filled operand times an infinity)
                const uint32_t pcol = col0 + pc * PIECE;
                if (ep.bias_on_rows) {
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) row_sum += pcol + j < p.N ? v[j] : 0.f;
                } else {
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) v[j] = row < end ? v[j] : 0.f;
                    const float    sum   = warp_column_sums(v, lane);
                    const uint32_t block = ep.ragged == RAGGED_ROWS
                                               ? group_first_block(c.first, c.group, 32u) + (row0 - c.first) / 32u
                                               : c.z_out * ep.part_blocks + row0 / 32u;
                    if (lane < PIECE && pcol + lane < p.N) ep.part[static_cast<uint64_t>(block) * p.N + pcol + lane] = sum;
                }
            }
        }
        if (ep.part && ep.bias_on_rows && row < end)
            ep.part[(static_cast<uint64_t>(c.z_out) * ep.part_blocks + col0 / CH) * p.M + row] = row_sum;
        store(c, row0, col0, end, sbuf, xbuf);
        return true;
    }

    // After a give-up: the loads still in flight must land before this CTA's memory goes away.
    __device__ __forceinline__ void drain()
    {
        if (lane == 0) {
            for (uint32_t b = 0; b < 2u; ++b) {
                if (!((in_flight >> b) & 1u)) continue;
                const uint64_t t0 = ptx::global_timer_ns();
                while (!ptx::mbar_try_wait(in_bar + 8u * b, (in_phase >> b) & 1u)) {
                    if (ptx::global_timer_ns() - t0 > WAIT_LIMIT_NS) {
                        atomicOr(p.status, ST_DRAIN_WAIT);
                        break;
                    }
                }
            }
            ptx::tma_store_wait_read<0>();
        }
    }
};

// The transposing epilogue's part of a tile with an epilogue: a piece of `n` <= 16 columns from col0
// on of kernel row i (this lane's), D(i, j) lying at out[j * M + i].  `side`: the read matrix's values.
template <int OUT>
struct EpilogueColumns {
    using T = OutType<OUT>;
    const GemmParams&     p;
    const EpilogueParams& ep;
    uint32_t              lane;

    __device__ __forceinline__ uint64_t at(const WorkCoord& c, uint32_t col, uint32_t i) const
    {
        return (static_cast<uint64_t>(c.z_out) * p.N + col) * p.M + i;
    }

    __device__ __forceinline__ void load_side(const WorkCoord& c, uint32_t col0, uint32_t n, uint32_t i, bool live, float (&side)[PIECE]) const
    {
        const T* src = static_cast<const T*>(ep.gradient ? ep.preact : ep.residual);
#pragma unroll
        for (uint32_t r = 0; r < PIECE; ++r) side[r] = live && r < n ? to_f32(src[at(c, col0 + r, i)]) : 0.f;
    }

    // Bias gradients: the piece's sum over the columns is added to `row_sum`, its sums over the rows go
    // to row `block_rows` of the partial sums.
    __device__ __forceinline__ void finish(const WorkCoord& c, uint32_t col0, uint32_t n, uint32_t i, bool live, uint32_t block_rows,
                                           float (&v)[PIECE], const float (&side)[PIECE], float& row_sum) const
    {
        if (ep.gradient) {
            if (ep.streamed)
                apply_slope(ep, v, side);
        } else {
            if (ep.bias) {
                const T* bias = static_cast<const T*>(ep.bias) + (ep.ragged == RAGGED_ROWS ? c.group : c.z_in) * ep.bias_stride;
                if (ep.bias_on_rows) {
                    const float b = live ? to_f32(bias[i]) : 0.f;
#pragma unroll
                    for (int r = 0; r < PIECE; ++r) v[r] += b;
                } else {
#pragma unroll
                    for (uint32_t r = 0; r < PIECE; ++r) v[r] += r < n ? to_f32(bias[col0 + r]) : 0.f;
                }
            }
            if (ep.aux && live) {
                T* pre = static_cast<T*>(ep.preact);
#pragma unroll
                for (uint32_t r = 0; r < PIECE; ++r)
                    if (r < n) pre[at(c, col0 + r, i)] = from_f32<T>(v[r]);
            }
            apply_activation(ep, v);
            if (ep.streamed) add_values(v, side);
        }
        if (live) {
            T* out = static_cast<T*>(p.out);
#pragma unroll
            for (uint32_t r = 0; r < PIECE; ++r)
                if (r < n) out[at(c, col0 + r, i)] = from_f32<T>(v[r]);
        }
        if (!ep.part) return;
        if (ep.bias_on_rows) {
#pragma unroll
            for (uint32_t r = 0; r < PIECE; ++r) row_sum += r < n ? v[r] : 0.f;
        } else {
#pragma unroll
            for (int r = 0; r < PIECE; ++r) v[r] = live ? v[r] : 0.f;
            const float sum = warp_column_sums(v, lane);
            if (lane < n) ep.part[static_cast<uint64_t>(block_rows) * p.N + col0 + lane] = sum;
        }
    }

    // A chunk of up to 32 columns from col0 on, `n` of them live.  `side`: the read values of the first
    // piece, loaded before the accumulator was awaited.
    template <class Pieces, class F>
    __device__ __forceinline__ void chunk(const WorkCoord& c, uint32_t col0, uint32_t n, uint32_t i, bool live, uint32_t block,
                                          uint32_t block_rows, Pieces& pieces, uint32_t npieces, float (&side)[PIECE], F&& accumulators_read) const
    {
        float row_sum = 0.f;
#pragma unroll 1
        for (uint32_t pc = 0; pc < npieces; ++pc) {
            const uint32_t m = n > pc * PIECE ? min(n - pc * PIECE, static_cast<uint32_t>(PIECE)) : 0u;
            float          v[PIECE];
            if (pc > 0u && ep.streamed) load_side(c, col0 + pc * PIECE, m, i, live, side);
            pieces.get(pc, v, accumulators_read);
            if (m) finish(c, col0 + pc * PIECE, m, i, live, block_rows, v, side, row_sum);
        }
        if (ep.part && ep.bias_on_rows && live && n) ep.part[static_cast<uint64_t>(block) * p.M + i] = row_sum;
    }
};

// One epilogue warp of the pair kernel with the transposing epilogue: chunks of 32 columns (of C's rows)
// from col0 on by the 32 kernel rows from row0 on (one per lane; contiguous in C), staged as 32 lines
// of 32 elements (no swizzle: a warp's accesses are whole lines), which TMA moves from and to C and the
// matrices like it.  A bias is one value per lane, its gradient a sum over a lane's registers.  Ragged
// rows only.
template <int OUT>
struct EpilogueTransposed {
    using T = OutType<OUT>;
    static constexpr uint32_t LINE = 32u * sizeof(T), BUF = 32u * LINE;

    const GemmParams&     p;
    const EpilogueParams& ep;
    const EpilogueMaps&   em;
    const CUtensorMap&    tmD;
    uint32_t              lane;
    uint32_t              stg;    // staging buffers: ep.bufs for C, then one for Z
    uint32_t              in_bar; // barriers of the first two
    volatile uint32_t*    s_abort;
    uint32_t              count     = 0; // as in EpilogueWarp
    uint32_t              in_phase  = 0;
    uint32_t              in_flight = 0;

    __device__ __forceinline__ uint32_t slot(uint32_t k) const { return (count + k) & (ep.bufs - 1u); }

    __device__ __forceinline__ void request(uint32_t k, uint32_t row0, uint32_t col0)
    {
        const uint32_t b = slot(k);
        if (lane == 0) {
            ptx::mbar_expect_tx(in_bar + 8u * b, BUF);
            ptx::tma_load_3d(stg + b * BUF, &em.in, in_bar + 8u * b, row0, col0, 0, 0);
        }
        in_flight |= 1u << b;
    }

    __device__ __forceinline__ void buffers_free()
    {
        ptx::fence_proxy_async_smem();
        if (lane == 0) ptx::tma_store_wait_read<0>();
        __syncwarp();
    }

    __device__ __forceinline__ float row_bias(const WorkCoord& c, uint32_t row) const
    {
        if (!ep.bias || row >= p.M) return 0.f;
        return to_f32(static_cast<const T*>(ep.bias)[c.group * ep.bias_stride + row]);
    }

    // Columns [col0, min(col0 + 32, stop)) are the group's.  False: a wait ran out.
    template <class F>
    __device__ __forceinline__ bool chunk(const WorkCoord& c, uint32_t row0, uint32_t col0, uint32_t stop, float bias, TmemPieces& pieces, F&& accumulators_read)
    {
        const uint32_t b    = slot(0);
        const uint32_t sbuf = stg + b * BUF, xbuf = stg + ep.bufs * BUF, at = lane * static_cast<uint32_t>(sizeof(T));
        if (ep.streamed) {
            bool ok = bounded_wait(in_bar + 8u * b, (in_phase >> b) & 1u, s_abort, p.status, ST_EPI_WAIT);
            ok      = __all_sync(0xffffffffu, ok);
            if (!ok) return false;
            in_phase ^= 1u << b;
            in_flight &= ~(1u << b);
        }
        // the buffers written below must have been read by the stores that last used them
        if (lane == 0) {
            if (ep.aux || ep.bufs == 1u) ptx::tma_store_wait_read<0>();
            else if (!ep.streamed) ptx::tma_store_wait_read<1>();
        }
        __syncwarp();
        float row_sum = 0.f;
#pragma unroll 1
        for (uint32_t pc = 0; pc < 32u / PIECE; ++pc) {
            const uint32_t first = pc * PIECE, to = sbuf + first * LINE + at;
            float          v[PIECE], side[PIECE];
            pieces.get(pc, v, accumulators_read);
            if (ep.streamed)
#pragma unroll
                for (uint32_t j = 0; j < PIECE; ++j) side[j] = to_f32(ld_shared_elem<T>(to + j * LINE));
            if (ep.gradient) {
                if (ep.streamed) apply_slope(ep, v, side);
            } else {
                if (ep.bias)
#pragma unroll
                    for (uint32_t j = 0; j < PIECE; ++j) v[j] += bias;
                if (ep.aux)
#pragma unroll
                    for (uint32_t j = 0; j < PIECE; ++j) st_shared_elem(xbuf + (first + j) * LINE + at, from_f32<T>(v[j]));
                apply_activation(ep, v);
                if (ep.streamed) add_values(v, side);
            }
#pragma unroll
            for (uint32_t j = 0; j < PIECE; ++j) st_shared_elem(to + j * LINE, from_f32<T>(v[j]));
            if (ep.part)
#pragma unroll
                for (uint32_t j = 0; j < PIECE; ++j) row_sum += col0 + first + j < stop ? v[j] : 0.f;
        }
        const uint32_t row = row0 + lane;
        if (ep.part && row < p.M)
            ep.part[(static_cast<uint64_t>(group_first_block(c.first, c.group, 32u)) + (col0 - c.first) / 32u) * p.M + row] = row_sum;
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (col0 + 32u <= stop) {
            if (lane == 0) {
                ptx::tma_store_3d(&tmD, sbuf, row0, col0, 0, 0);
                if (ep.aux) ptx::tma_store_3d(&em.aux, xbuf, row0, col0, 0, 0);
            }
        } else if (row < p.M) { // the lines from `stop` on are the next group's
            const uint64_t to = static_cast<uint64_t>(col0) * p.M + row;
            for (uint32_t j = 0; j < stop - col0; ++j) {
                static_cast<T*>(p.out)[to + static_cast<uint64_t>(j) * p.M] = ld_shared_elem<T>(sbuf + j * LINE + at);
                if (ep.aux) static_cast<T*>(ep.preact)[to + static_cast<uint64_t>(j) * p.M] = ld_shared_elem<T>(xbuf + j * LINE + at);
            }
        }
        if (lane == 0) ptx::tma_store_commit(); // (an empty group keeps the count of the waits)
        __syncwarp();
        ++count;
        return true;
    }

    // After a give-up: the loads still in flight must land before this CTA's memory goes away.
    __device__ __forceinline__ void drain()
    {
        if (lane == 0) {
            for (uint32_t b = 0; b < 2u; ++b) {
                if (!((in_flight >> b) & 1u)) continue;
                const uint64_t t0 = ptx::global_timer_ns();
                while (!ptx::mbar_try_wait(in_bar + 8u * b, (in_phase >> b) & 1u)) {
                    if (ptx::global_timer_ns() - t0 > WAIT_LIMIT_NS) {
                        atomicOr(p.status, ST_DRAIN_WAIT);
                        break;
                    }
                }
            }
            ptx::tma_store_wait_read<0>();
        }
    }
};

template <int BN, int OUT, int CL, bool TR, bool GATHER, bool KS = false, bool EP = false>
__device__ __forceinline__ void gemm_umma_body(const CUtensorMap& tmA, const CUtensorMap& tmB,
                                               const CUtensorMap* tmDs, const CUtensorMap& tmW, const GemmParams& p,
                                               const EpilogueMaps* em = nullptr, const EpilogueParams* epp = nullptr)
{
    const CUtensorMap& tmD = tmDs[0];
    static_assert(BN == 16 || BN == 32 || BN == 64 || BN == 128 || BN == 256 || BN == 512,
                  "BN must be 16, 32, 64, 128, 256 or 512");
    static_assert(CL == 1 || CL == 2, "cluster size must be 1 or 2");
    static_assert(!TR || CL == 1 || (EP && BN == 256), "the transposed epilogue: one-CTA kernels, and the pair kernel of ragged rows");
    constexpr bool TRP = TR && CL == 2; // ragged rows along N, tiles of equal width per group, a staged transposing epilogue
    static_assert(!KS || (CL == 1 && !GATHER && ((!TR && BN >= 128 && BN <= 256) || (TR && BN <= 128))),
                  "cluster K partitions: one-CTA staged tiles of 128 or 256 columns, transposed slabs of up to 128");
    // One MMA covers at most 256 columns: a 512-wide tile is two sub-tiles that share the A'
    // operand of every K slice (A' is staged once for 512 columns of output).
    constexpr int      UMMA_N       = BN > 256 ? 256 : BN;
    constexpr int      NSUB         = BN / UMMA_N;
    constexpr int      SUB_ROWS     = UMMA_N / CL;          // B' rows per sub-tile in this CTA
    constexpr int      BN_CTA       = NSUB * SUB_ROWS;      // B' rows this CTA stages
    constexpr uint32_t SUB_BYTES    = SUB_ROWS * BLOCK_K * 2;
    constexpr uint32_t B_TILE_BYTES = BN_CTA * BLOCK_K * 2;
    constexpr uint32_t STAGE_BYTES  = A_TILE_BYTES + B_TILE_BYTES;
    // TMEM holds 512 f32 columns: two accumulators (epilogue of tile i overlaps the main loop
    // of tile i + 1) up to BN = 256, a single one for BN = 512.
    constexpr uint32_t NUM_ACC      = BN > 256 ? 1 : 2;
    constexpr uint32_t ACC_COLS     = BN < 64 ? 64 : BN; // the epilogue reads up to 64 columns at a time
    constexpr uint32_t TMEM_COLS    = NUM_ACC * ACC_COLS; // power of two >= 32
    constexpr int      OUT_BYTES    = (OUT == OUT_F32) ? 4 : 2;
    constexpr int      CH           = 128 / OUT_BYTES; // output columns per 128-byte chunk
    constexpr int      NCHUNK       = BN < CH ? 1 : BN / CH; // a narrow tile is one (clipped) chunk
    static_assert(SUB_ROWS >= 16, "each CTA stages at least 16 rows of B' per sub-tile");
    // (an MN-major B' is loaded in 64-row boxes: the host only picks BN >= 64 * CL for it)

#ifdef B200_GEMM_TIMELINE
    __shared__ uint32_t s_tl_base;
    if (blockIdx.x == 0 && threadIdx.x == 0) s_tl_base = (atomicAdd(&g_timeline_count, 1u) % TIMELINE_ROWS) * TIMELINE_SLOTS;
    uint32_t tl_base = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        tl_base = s_tl_base;
        B200_TLG(0);
        B200_TL(1);
    }
#endif
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_full[TR ? MAX_SLAB_STAGES : MAX_STAGES];
    __shared__ __align__(8) uint64_t s_empty[TR ? MAX_SLAB_STAGES : MAX_STAGES];
    __shared__ __align__(8) uint64_t s_tfull[2];
    __shared__ __align__(8) uint64_t s_tempty[2];
    __shared__ __align__(8) uint64_t s_drain;
    __shared__ uint32_t              s_tmem_base;
    __shared__ volatile uint32_t     s_abort;
    static_assert(!EP || !GATHER, "no gathering kernels with an epilogue");
    constexpr int                    EPW = EP ? EPI_WARPS : 4; // epilogue warps
    __shared__ volatile uint32_t     s_seen[2];                                          // EP: the accumulator awaited last is complete
    __shared__ __align__(8) uint64_t s_in[EP && (!TR || CL == 2) ? EPI_WARPS * 2 : 1];                // EP: chunk of the read matrix landed
    constexpr uint32_t               BIAS_BYTES = (UMMA_N < 32 * EPI_WARPS ? 32 * EPI_WARPS : UMMA_N) * OUT_BYTES;
    __shared__ __align__(16) uint8_t s_bias[EP && !TR ? 2 * BIAS_BYTES : 16];            // EP: a tile's biases, two tiles in turn

    const uint32_t tid    = threadIdx.x;
    const uint32_t warp   = tid >> 5;
    const uint32_t lane   = tid & 31u;
    const uint32_t stages = p.stages;
    const uint32_t rank   = (CL == 2) ? ptx::cluster_ctarank() : 0u; // CTA rank in the pair
    // KS: the cluster is the worker, its rank the K partition (p.split_k CTAs per cluster).
    const uint32_t krank  = KS ? ptx::cluster_ctarank() : 0u;
    const uint32_t unit   = KS ? blockIdx.x / p.split_k : blockIdx.x / CL; // persistent worker index
    const uint32_t units  = KS ? gridDim.x / p.split_k : gridDim.x / CL;
    WorkCoord      ks_c{};        // KS: the one tile of this cluster (epilogue warps)
    bool           ks_ok = false; // KS: accumulator complete

    // Bytes of A' per ring slot and slot pitch: compile-time for the staged epilogue; the
    // transposed variant stages p.bm (a multiple of 8, <= 128) rows of A' per slot.
    // One-CTA kernels up to 256 columns use "slots" of kc k-blocks:
    // [A' k-block 0 .. kc-1][B' k-block 0 .. kc-1], each operand fetched by one TMA instruction
    // (the per-slot barrier and issue work of the two single-thread roles is amortised over kc
    // k-blocks; with narrow tiles that work, not the tensor pipe, bounds the K loop).  A' has
    // p.bm rows per k-block: 128, or a shorter slab with the transposed epilogue.
    constexpr bool SLOT    = (CL == 1) && (NSUB == 1);
    const uint32_t kc      = SLOT ? p.kc : 1u;
    const uint32_t a_bytes = SLOT ? p.bm * (BLOCK_K * 2u) : A_TILE_BYTES;
    const uint32_t pitch   = SLOT ? kc * (a_bytes + B_TILE_BYTES) : STAGE_BYTES;
    const uint32_t tile_m  = SLOT ? p.bm : static_cast<uint32_t>(BLOCK_M * CL);
    // CTA-pair kernels up to 256 columns take the tile width at run time (any multiple of the
    // epilogue's 128-byte chunk up to BN): the MMA's N extent is a field of the instruction
    // descriptor and the B' box height a field of the tensor map, so one compiled kernel serves
    // widths that cut N into whole waves of tiles.  Ring slots and TMEM stay sized for BN.
    constexpr bool FLEX     = (CL == 2) && (NSUB == 1);
    const uint32_t wn       = FLEX ? p.wn : static_cast<uint32_t>(BN);
    const uint32_t sub_rows = FLEX ? wn / CL : static_cast<uint32_t>(SUB_ROWS);
    const uint32_t sub_bytes = FLEX ? sub_rows * (BLOCK_K * 2u) : SUB_BYTES;

    const uint32_t ring = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u; // ring of operand tiles
    const uint32_t epi  = ring + stages * pitch;                      // epilogue staging (unused when TR)
    GroupTable     gt{nullptr, nullptr};
    if constexpr (EP) { // the group table lies at the very end of the dynamic shared memory
        if (epp->ragged != RAGGED_NONE) {
            uint32_t* tab = reinterpret_cast<uint32_t*>(smem_raw + epp->table_at);
            gt.first      = tab;
            gt.tiles      = tab + epp->groups + 1u;
            if (warp == 2) {
                ptx::grid_dep_wait(); // the offsets may come from the kernel before this one
                build_group_table(*epp, TR ? static_cast<uint32_t>(BN) : tile_m, tab, tab + epp->groups + 1u);
            }
        }
    }
    auto next_work = [&](WorkCursor& cur, WorkCoord& c) -> bool {
        if constexpr (EP) return work_next_epilogue<TR, TRP>(p, *epp, gt, cur, units, wn, tile_m, c);
        else return work_next(p, cur, unit, units, wn, tile_m, c);
    };

    if (warp == 0) {
        // Barrier set-up spread over the lanes of warp 0 (one thread doing all of it serially is
        // a third of a microsecond of every launch; small problems notice).
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmA);
            ptx::prefetch_tensormap(&tmB);
            if constexpr (GATHER) {
                for (uint32_t d = 0; d < p.ndst; ++d) ptx::prefetch_tensormap(&tmDs[d]);
            } else {
                ptx::prefetch_tensormap(&tmD);
            }
            ptx::mbar_init(ptx::smem_u32(&s_drain), 1);
            s_abort = 0u;
        }
        if (lane < stages) {
            ptx::mbar_init(ptx::smem_u32(&s_full[lane]), 1);
            ptx::mbar_init(ptx::smem_u32(&s_empty[lane]), 1);
        }
        if (lane >= 30u) {
            ptx::mbar_init(ptx::smem_u32(&s_tfull[lane - 30u]), 1);
            ptx::mbar_init(ptx::smem_u32(&s_tempty[lane - 30u]), EPW * CL);
        }
        if constexpr (EP && (!TR || TRP)) {
            if (lane < EPI_WARPS * 2) ptx::mbar_init(ptx::smem_u32(&s_in[lane]), 1);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<CL>(ptx::smem_u32(&s_tmem_base), TMEM_COLS);
    }
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (CL == 2) { // the peer's barriers must exist before anything arrives on them
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    ptx::tc_fence_after();
#ifdef B200_GEMM_TIMELINE
    tl_base = s_tl_base;
    if (threadIdx.x == 0) B200_TL(2);
#endif
    const uint32_t tmem_base = s_tmem_base;
    // Programmatic dependent launch, both directions.  This grid may have been scheduled while
    // the kernel before it in the stream was still draining: everything above touched only this
    // CTA's shared memory and TMEM.  Each thread that touches global memory waits for the kernel
    // before this one right before its first access (the producer before its first TMA load, the
    // epilogue threads before their first store), so the work decode, the address arithmetic and
    // the first barrier operations of every role run while that kernel drains - about a
    // microsecond of every launch otherwise.  The MMA thread touches no global memory.  The
    // kernel after this one (a reduction pass, or the next GEMM) may be scheduled as SMs free
    // up; it waits for this grid to complete before it reads or writes anything.
    ptx::grid_dep_launch();
    bool dep_waited = false;
    auto dep_wait = [&]() {
        if (!dep_waited) {
            ptx::grid_dep_wait();
            dep_waited = true;
        }
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        if (ptx::elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0;
            bool     ok = true;
            const uint64_t pol_a = ptx::make_l2_policy(p.l2_hints & 3u);
            const uint64_t pol_b = ptx::make_l2_policy((p.l2_hints >> 2) & 3u);
            WorkCursor cur = work_begin(p, unit, krank);
            WorkCoord  c;
            const CUtensorMap* mapA = &tmA;
            const CUtensorMap* mapB = &tmB;
            for (uint32_t w = unit; ok && next_work(cur, c); w += units) {
                if constexpr (EP) {
                    if (epp->ragged == RAGGED_K && c.kb1 > c.kb0 && mapA != epp->maps + 2u * c.group) {
                        mapA = epp->maps + 2u * c.group; // this group's own maps, written by the kernel before this one
                        mapB = mapA + 1;
                        dep_wait();
                        ptx::fence_tensormap_acquire(mapA);
                        ptx::fence_tensormap_acquire(mapB);
                    }
                } else {
                    c.z_a = c.z_b = c.z_in;
                    c.k_first = 0u;
                }
                const int32_t   am = static_cast<int32_t>(c.m0 + rank * BLOCK_M);
                const int32_t   bn = static_cast<int32_t>(c.n0 + rank * (TRP ? c.wn / 2u : sub_rows));
                // Streaming (HBM-bound) problems rotate each work unit's K order so that the CTAs
                // running at the same time read different K offsets: rows of a K-major operand
                // are a power of two apart, and same-offset reads from thousands of rows land on
                // a few memory channels.
                const uint32_t nkb = c.kb1 - c.kb0;
                if constexpr (SLOT) {
                    // One slot = kc k-blocks of A' (p.bm rows) and of B' (BN rows),
                    // one TMA instruction per operand (per 64-row half for an MN-major operand).
                    // Boxes that reach past K read zeros, so a ragged last slot needs no care.
                    // Two cluster K partitions are interleaved: rank r takes the ring-slot-sized K
                    // steps r, r + 2, r + 4, ... so that the two CTAs, which run in step, read
                    // neighbouring pieces of the same operand rows at the same time.  (Measured
                    // 1 - 5 % faster than two contiguous halves on 128x8192x8192; four interleaved
                    // partitions measured 8 % slower than four contiguous quarters.)
                    const bool     ileave = KS && p.split_k == 2u;
                    const uint32_t nst  = ileave ? ((p.k_blocks + kc - 1u) / kc + 1u - krank) / 2u : (nkb + kc - 1u) / kc;
                    const uint32_t rot  = (p.k_skew && nst) ? static_cast<uint32_t>((static_cast<uint64_t>(w) * p.k_skew) % nst) : 0u;
                    const uint32_t half = kc * (64u * BLOCK_K * 2u); // bytes of one 64-row half of an MN-major operand
                    for (uint32_t i = 0; i < nst; ++i) {
                        const uint32_t rel = i + rot >= nst ? i + rot - nst : i + rot;
                        const int32_t  kb  = ileave ? static_cast<int32_t>((krank + rel * 2u) * kc)
                                                    : static_cast<int32_t>(c.kb0 + rel * kc);
                        const int32_t  k0  = kb * BLOCK_K + static_cast<int32_t>(c.k_first);
                        ok = bounded_wait(ptx::smem_u32(&s_empty[stage]), phase ^ 1u, &s_abort,
                                          p.status, ST_PRODUCER_WAIT);
                        if (!ok) break;
                        const uint32_t sa  = ring + stage * pitch;
                        const uint32_t sb  = sa + kc * a_bytes;
                        const uint32_t bar = ptx::smem_u32(&s_full[stage]);
                        ptx::mbar_expect_tx(bar, pitch);
                        if (issued == 0) B200_TLG(15);
                        dep_wait();
                        if (issued == 0) {
                            B200_TL(3);
                            B200_TL_CTA(0);
                        }
                        if (p.a_mn_major == 0u) {
                            if (p.k4d) ptx::tma_load_4d(sa, mapA, bar, 0, am, kb, c.z_a, pol_a);
                            else ptx::tma_load_3d(sa, mapA, bar, k0, am, c.z_a, pol_a);
                        } else {
                            ptx::tma_load_3d(sa, mapA, bar, am, k0, c.z_a, pol_a);
                            if (p.bm > 64u) ptx::tma_load_3d(sa + half, mapA, bar, am + 64, k0, c.z_a, pol_a);
                        }
                        if (p.b_mn_major == 0u) {
                            if (p.k4d) ptx::tma_load_4d(sb, mapB, bar, 0, bn, kb, c.z_b, pol_b);
                            else ptx::tma_load_3d(sb, mapB, bar, k0, bn, c.z_b, pol_b);
                        } else {
#pragma unroll
                            for (int j = 0; j < SUB_ROWS / 64; ++j)
                                ptx::tma_load_3d(sb + j * half, mapB, bar, bn + j * 64, k0, c.z_b, pol_b);
                        }
                        if (issued == 0) B200_TL(4);
                        ++issued;
                        B200_TL(5);
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    continue;
                }
                const uint32_t rot = p.k_skew ? static_cast<uint32_t>((static_cast<uint64_t>(w) * p.k_skew) % nkb) : 0u;
                const uint32_t stg_x  = (NSUB == 2) ? min(p.stagger, nkb) : 0u;
                const uint32_t nsteps = nkb + stg_x;
                for (uint32_t i = 0; i < nsteps; ++i) {
                    const TileStep ts   = (NSUB == 2) ? tile_step(i, nkb, stg_x) : TileStep{i, 1u};
                    const uint32_t rel  = ts.kb_rel + rot >= nkb ? ts.kb_rel + rot - nkb : ts.kb_rel + rot;
                    const uint32_t kb   = c.kb0 + rel;
                    const uint32_t nsub = (NSUB == 2) ? __popc(ts.mask) : 1u;
                    ok = bounded_wait(ptx::smem_u32(&s_empty[stage]), phase ^ 1u, &s_abort,
                                      p.status, ST_PRODUCER_WAIT);
                    if (!ok) break;
                    const uint32_t sa = ring + stage * pitch;
                    const uint32_t sb = sa + a_bytes;
                    const int32_t  k0 = static_cast<int32_t>(kb * BLOCK_K + c.k_first);
                    const uint32_t step_bytes = a_bytes + nsub * sub_bytes; // this CTA's share
                    uint32_t       bar = ptx::smem_u32(&s_full[stage]);
                    if constexpr (CL == 2) {
                        // Rank 0 owns the pair's full barrier and expects both CTAs' bytes.
                        if (rank == 0) ptx::mbar_expect_tx(bar, 2 * step_bytes);
                        bar = ptx::mapa_u32(bar, 0);
                    } else {
                        ptx::mbar_expect_tx(bar, step_bytes);
                    }
                    if (issued == 0) B200_TLG(15);
                    dep_wait();
                    if (issued == 0) {
                        B200_TL(3);
                        B200_TL_CTA(0);
                    }
                    if (p.a_mn_major == 0u) {
                        tma_load<CL>(sa, mapA, bar, k0, am, c.z_a, pol_a);
                    } else if (EP && CL == 2 && epp->whole_a) {
                        ptx::tma_load_4d_pair(sa, mapA, bar, 0, k0, am / 64, c.z_a);
                    } else {
#pragma unroll
                        for (int j = 0; j < BLOCK_M / 64; ++j)
                            tma_load<CL>(sa + j * (64 * BLOCK_K * 2), mapA, bar, am + j * 64, k0,
                                         c.z_a, pol_a);
                    }
#pragma unroll
                    for (int h = 0; h < NSUB; ++h) {
                        if (NSUB == 2 && !((ts.mask >> h) & 1u)) continue;
                        const int32_t  bh = bn + h * UMMA_N; // first B' row of sub-tile h
                        const uint32_t sh = sb + h * SUB_BYTES;
                        if (p.b_mn_major == 0u) {
                            tma_load<CL>(sh, mapB, bar, k0, bh, c.z_b, pol_b);
                        } else if (EP && CL == 2 && epp->whole_b) {
                            ptx::tma_load_4d_pair(sh, mapB, bar, 0, k0, bh / 64, c.z_b);
                        } else {
#pragma unroll
                            for (int j = 0; j < SUB_ROWS / 64; ++j)
                                if (!FLEX || static_cast<uint32_t>(j) * 64u < sub_rows)
                                    tma_load<CL>(sh + j * (64 * BLOCK_K * 2), mapB, bar, bh + j * 64,
                                                 k0, c.z_b, pol_b);
                        }
                    }
                    if (issued == 0) B200_TL(4);
                    ++issued;
                    B200_TL(5);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (s_abort != 0u && rank == 0) {
                // Gave up somewhere: let the loads already in flight land before the CTA exits.
                const uint32_t pending = min(issued, stages);
                for (uint32_t i = 0; i < pending; ++i) {
                    if (stage == 0) {
                        stage = stages;
                        phase ^= 1u;
                    }
                    --stage;
                    const uint64_t t0 = ptx::global_timer_ns();
                    while (!ptx::mbar_try_wait(ptx::smem_u32(&s_full[stage]), phase)) {
                        if (ptx::global_timer_ns() - t0 > WAIT_LIMIT_NS) {
                            atomicOr(p.status, ST_DRAIN_WAIT);
                            break;
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (ptx::elect_one() && rank == 0) {
            // K-major swizzled tiles ignore the leading offset (canonical value: 16 bytes).
            const uint32_t a_lbo   = p.a_mn_major ? 64u * BLOCK_K * 2u : 16u;
            const uint32_t b_lbo   = p.b_mn_major ? 64u * BLOCK_K * 2u : 16u;
            // Descriptor start-address step (16-byte units) per K = 16 slice.
            const uint32_t a_kstep = p.a_mn_major ? (2u * 1024u) >> 4 : (UMMA_K * 2u) >> 4;
            const uint32_t b_kstep = p.b_mn_major ? (2u * 1024u) >> 4 : (UMMA_K * 2u) >> 4;
            uint32_t       stage = 0, phase = 0, it = 0;
            bool           ok = true;
            WorkCursor cur = work_begin(p, unit, krank);
            WorkCoord  c;
            for (; ok && next_work(cur, c); ++it) {
                if constexpr (NSUB == 2) {
                    // Two column halves with their own full / empty barriers (s_tfull[h],
                    // s_tempty[h]), staggered by stg_x k-blocks: see TileStep.  Three
                    // straight-line loops (half 0 alone, both, half 1 alone): the MMAs of one
                    // step must be issued back to back, with no branch between the two halves
                    // that share an A' tile — a conditional in this loop costs 10 % of the
                    // kernel's throughput.
                    const uint32_t nkb    = c.kb1 - c.kb0;
                    const uint32_t stg_x  = min(p.stagger, nkb);
                    const uint32_t tphase = it & 1u;
                    auto step = [&](auto mask_c, uint32_t acc0, uint32_t acc1) -> bool {
                        constexpr uint32_t MASK = decltype(mask_c)::value;
                        if (!bounded_wait(ptx::smem_u32(&s_full[stage]), phase, &s_abort, p.status,
                                          ST_MMA_WAIT_FULL))
                            return false;
                        ptx::tc_fence_after();
                        const uint32_t sa = ring + stage * pitch;
                        const uint32_t sb = sa + a_bytes;
                        const uint64_t ad = ptx::make_smem_desc(sa, a_lbo, 1024u);
                        const uint64_t bd = ptx::make_smem_desc(sb, b_lbo, 1024u);
#pragma unroll
                        for (uint32_t k = 0; k < BLOCK_K / UMMA_K; ++k) {
                            if constexpr ((MASK & 1u) != 0u)
                                ptx::umma_f16<CL>(tmem_base, ad + k * a_kstep, bd + k * b_kstep, p.idesc,
                                                  (acc0 | k) ? 1u : 0u);
                            if constexpr ((MASK & 2u) != 0u)
                                ptx::umma_f16<CL>(tmem_base + UMMA_N, ad + k * a_kstep,
                                                  bd + (SUB_BYTES >> 4) + k * b_kstep, p.idesc,
                                                  (acc1 | k) ? 1u : 0u);
                        }
                        umma_arrive<CL>(ptx::smem_u32(&s_empty[stage]));
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                        return true;
                    };
                    // half 0 starts: its columns must have been drained
                    ok = bounded_wait<CL == 2>(ptx::smem_u32(&s_tempty[0]), tphase ^ 1u, &s_abort, p.status,
                                               ST_MMA_WAIT_ACC);
                    for (uint32_t i = 0; ok && i < stg_x; ++i)
                        ok = step(std::integral_constant<uint32_t, 1u>{}, i > 0u ? 1u : 0u, 0u);
                    if (!ok) break;
                    // half 1 starts
                    ok = bounded_wait<CL == 2>(ptx::smem_u32(&s_tempty[1]), tphase ^ 1u, &s_abort, p.status,
                                               ST_MMA_WAIT_ACC);
                    for (uint32_t i = stg_x; ok && i < nkb; ++i)
                        ok = step(std::integral_constant<uint32_t, 3u>{}, i > 0u ? 1u : 0u, i > stg_x ? 1u : 0u);
                    if (!ok) break;
                    umma_arrive<CL>(ptx::smem_u32(&s_tfull[0])); // half 0 complete
                    for (uint32_t i = 0; ok && i < stg_x; ++i)
                        ok = step(std::integral_constant<uint32_t, 2u>{}, 0u, (nkb > stg_x || i > 0u) ? 1u : 0u);
                    if (!ok) break;
                    umma_arrive<CL>(ptx::smem_u32(&s_tfull[1])); // half 1 complete
                    B200_TL(7);
                    continue;
                }
                const uint32_t buf    = it % NUM_ACC;
                const uint32_t aphase = (it / NUM_ACC) & 1u;
                ok = bounded_wait<CL == 2>(ptx::smem_u32(&s_tempty[buf]), aphase ^ 1u, &s_abort,
                                           p.status, ST_MMA_WAIT_ACC);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint32_t d_tmem = tmem_base + buf * ACC_COLS;
                if constexpr (SLOT) {
                    // kc k-blocks per slot; see the producer for the slot layout.
                    const uint32_t nst    = (KS && p.split_k == 2u) ? ((p.k_blocks + kc - 1u) / kc + 1u - krank) / 2u // interleaved, see the producer
                                                                    : (c.kb1 - c.kb0 + kc - 1u) / kc;
                    const uint32_t half   = kc * (64u * BLOCK_K * 2u);
                    const uint32_t a_blk  = p.a_mn_major ? 64u * BLOCK_K * 2u : a_bytes;
                    const uint32_t b_blk  = p.b_mn_major ? 64u * BLOCK_K * 2u : B_TILE_BYTES;
                    const uint32_t a_lbo2 = p.a_mn_major ? half : 16u;
                    const uint32_t b_lbo2 = p.b_mn_major ? half : 16u;
                    for (uint32_t i = 0; i < nst; ++i) {
                        ok = bounded_wait(ptx::smem_u32(&s_full[stage]), phase, &s_abort, p.status,
                                          ST_MMA_WAIT_FULL);
                        if (!ok) break;
                        if (i == 0 && it == 0) B200_TL(6);
                        ptx::tc_fence_after();
                        const uint32_t sa = ring + stage * pitch;
                        const uint32_t sb = sa + kc * a_bytes;
                        for (uint32_t c2 = 0; c2 < kc; ++c2) {
                            const uint64_t ad = ptx::make_smem_desc(sa + c2 * a_blk, a_lbo2, 1024u);
                            const uint64_t bd = ptx::make_smem_desc(sb + c2 * b_blk, b_lbo2, 1024u);
#pragma unroll
                            for (uint32_t k = 0; k < BLOCK_K / UMMA_K; ++k) {
                                ptx::umma_f16<CL>(d_tmem, ad + k * a_kstep, bd + k * b_kstep, p.idesc,
                                                  (i | c2 | k) ? 1u : 0u);
                            }
                        }
                        umma_arrive<CL>(ptx::smem_u32(&s_empty[stage]));
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                } else {
                    // (bits 17 .. 22: the MMA's N extent / 8)
                    const uint32_t idesc = TRP ? (p.idesc & ~(0x3fu << 17)) | ((c.wn >> 3) << 17) : p.idesc;
                    for (uint32_t kb = c.kb0; kb < c.kb1; ++kb) {
                        ok = bounded_wait(ptx::smem_u32(&s_full[stage]), phase, &s_abort, p.status,
                                          ST_MMA_WAIT_FULL);
                        if (!ok) break;
                        if (kb == c.kb0 && it == 0) B200_TL(6);
                        ptx::tc_fence_after();
                        const uint32_t sa = ring + stage * pitch;
                        const uint32_t sb = sa + a_bytes;
                        const uint64_t ad = ptx::make_smem_desc(sa, a_lbo, 1024u);
                        const uint64_t bd = ptx::make_smem_desc(sb, b_lbo, 1024u);
#pragma unroll
                        for (uint32_t k = 0; k < BLOCK_K / UMMA_K; ++k) {
                            ptx::umma_f16<CL>(d_tmem, ad + k * a_kstep, bd + k * b_kstep, idesc,
                                              (kb > c.kb0 || k > 0u) ? 1u : 0u);
                        }
                        // Slot free (in both CTAs of a pair) once these MMAs retire.
                        umma_arrive<CL>(ptx::smem_u32(&s_empty[stage]));
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                if (!ok) break;
                umma_arrive<CL>(ptx::smem_u32(&s_tfull[buf])); // accumulator complete
                B200_TL(7);
            }
            // All MMAs must have retired before TMEM is released and shared memory goes away.
            if constexpr (CL == 2) ptx::umma_commit_pair(ptx::smem_u32(&s_drain), 0x1);
            else ptx::umma_commit(ptx::smem_u32(&s_drain));
            const uint64_t t0 = ptx::global_timer_ns();
            while (!ptx::mbar_try_wait(ptx::smem_u32(&s_drain), 0u)) {
                if (ptx::global_timer_ns() - t0 > WAIT_LIMIT_NS) {
                    atomicOr(p.status, ST_DRAIN_WAIT);
                    break;
                }
            }
            B200_TL(8);
        }
    } else if constexpr (EP) {
        // ------------------------------------------------------------------ epilogue with activation, bias, ...
        const uint32_t q  = warp & 3u;          // TMEM lane quarter this warp may read
        const uint32_t hw = (warp - 2u) >> 2;   // takes column chunks hw, hw + EPI_SETS, ...
        uint32_t       it = 0;
        bool           ok = true;
        WorkCursor     cur = work_begin(p, unit, krank);
        WorkCoord      c;
        auto release = [&](uint32_t bar_i) { // this warp has read its part of the accumulator
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CL == 2) ptx::mbar_arrive_cluster_relaxed(ptx::smem_u32(&s_tempty[bar_i]), 0);
                else ptx::mbar_arrive(ptx::smem_u32(&s_tempty[bar_i]));
            }
        };
        // One warp polls the accumulator's barrier, the others sleep at a named barrier: eight polling
        // warps took issue slots and power from the producer and MMA threads (4096 x 5120 x 5120 with a
        // residual 176 -> 164 us, the plain product 160).  Every warp calls this once per accumulator and
        // gets the same answer (s_seen alternates: the poller is at most one accumulator ahead).
        uint32_t waits = 0;
        auto accumulator = [&](uint32_t bar_i, uint32_t parity) -> bool {
            const uint32_t at = waits++ & 1u;
            if (warp == 2u) {
                const bool r = bounded_wait(ptx::smem_u32(&s_tfull[bar_i]), parity, &s_abort, p.status, ST_EPI_WAIT);
                const bool a = __all_sync(0xffffffffu, r);
                if (lane == 0) s_seen[at] = a ? 1u : 0u;
            }
            ptx::named_barrier(1u, 32u * EPI_WARPS);
            if (s_seen[at] == 0u) return false;
            (void)ptx::mbar_test_wait(ptx::smem_u32(&s_tfull[bar_i]), parity); // (completed: orders this warp behind it too)
            ptx::tc_fence_after();
            if (warp == 2u && lane == 0 && waits == 1u) {
                B200_TL(9);
                B200_TL_CTA(2);
            }
            return true;
        };
        [[maybe_unused]] uint32_t nstore = 0;
        auto stored = [&] { // (timeline) a chunk's stores have been issued
            if (warp == 2u && lane == 0) {
                if (nstore++ == 0u) B200_TL(10);
                B200_TL(11);
            }
        };
        if constexpr (KS) {
            // one tile per cluster; the partials are summed after the cluster barriers below
            if (next_work(cur, c)) {
                if constexpr (!TR) { // the tile's biases, for the sums after the cluster barriers
                    if (epp->bias && !epp->bias_on_rows && (warp - 2u) * 32u < static_cast<uint32_t>(BN)) {
                        dep_wait();
                        EpilogueWarp<OUT> ew{p, *epp, *em, tmD, p.out, lane, 0u, 0u, s_bias, &s_abort};
                        ew.fetch_bias(c, c.n0, (warp - 2u) * 32u, s_bias);
                    }
                }
                ok    = accumulator(0u, 0u);
                ks_c  = c;
                ks_ok = ok;
            }
        } else if constexpr (TRP) {
            using ET = EpilogueTransposed<OUT>;
            ET   et{p, *epp, *em, tmD, lane, epi + (warp - 2u) * (epp->bufs + epp->aux) * ET::BUF, ptx::smem_u32(&s_in[(warp - 2u) * 2u]), &s_abort};
            bool live_warp = true;
            for (; ok && next_work(cur, c); ++it) {
                const uint32_t buf  = it % NUM_ACC;
                const uint32_t row0 = c.m0 + rank * BLOCK_M + q * 32u;
                const uint32_t stop = min(c.end, c.n0 + c.wn);
                const uint32_t live = row0 < p.M && c.n0 < stop ? (stop - c.n0 + 31u) / 32u : 0u;
                const uint32_t mine = live > hw ? (live - hw + EPI_SETS - 1u) / EPI_SETS : 0u; // this warp's chunks: hw, hw + EPI_SETS, ...
                auto           col  = [&](uint32_t k) { return c.n0 + (hw + EPI_SETS * k) * 32u; };
                const uint32_t tacc = tmem_base + ((q * 32u) << 16) + buf * ACC_COLS;
                float          bias = 0.f;
                if (mine && live_warp) {
                    dep_wait();
                    if (epp->streamed) {
                        et.buffers_free();
                        for (uint32_t k = 0; k < min(epp->bufs, mine); ++k) et.request(k, row0, col(k));
                    }
                    bias = et.row_bias(c, row0 + lane);
                }
                ok = accumulator(buf, (it / NUM_ACC) & 1u);
                if (!ok) break;
                if (!live_warp) continue; // (it still meets the others at every accumulator)
                if (mine == 0u) release(buf);
#pragma unroll 1
                for (uint32_t k = 0; k < mine; ++k) {
                    TmemPieces pieces{tacc + (hw + EPI_SETS * k) * 32u, 32u / PIECE, c.kb1 == c.kb0};
                    if (epp->streamed && k > 0u && k - 1u + epp->bufs < mine) {
                        et.buffers_free(); // the chunk before this one left from the buffer asked for now
                        et.request(epp->bufs - 1u, row0, col(k - 1u + epp->bufs));
                    }
                    live_warp = et.chunk(c, row0, col(k), stop, bias, pieces, [&] { if (k + 1u == mine) release(buf); });
                    stored();
                    if (!live_warp) break; // (a wait ran out: the abort flag ends the other roles)
                }
            }
            et.drain();
        } else if constexpr (TR) {
            const EpilogueColumns<OUT> ec{p, *epp, lane};
            constexpr uint32_t         CHUNKS = (BN + 31) / 32;
            const uint32_t             bs     = BN < 32 ? BN : 32; // columns per block of sums
            for (; ok && next_work(cur, c); ++it) {
                const uint32_t buf  = it % NUM_ACC;
                const uint32_t i    = c.m0 + q * 32u + lane;
                const bool     live = (q * 32u + lane) < p.bm && i < p.M;
                const uint32_t tacc = tmem_base + ((q * 32u) << 16) + buf * ACC_COLS;
                bool           seen = false;
                dep_wait();
#pragma unroll 1
                for (uint32_t ch = hw; ch < CHUNKS; ch += EPI_SETS) {
                    const uint32_t col0 = c.n0 + ch * 32u;
                    const uint32_t n    = col0 < c.end ? min(min(32u, BN - ch * 32u), c.end - col0) : 0u;
                    constexpr uint32_t NP = (BN < 32 ? BN : 32) / PIECE; // pieces of a chunk
                    float          side[PIECE];
                    if (epp->streamed) ec.load_side(c, col0, min(n, static_cast<uint32_t>(PIECE)), i, live, side);
                    if (!seen) {
                        ok = accumulator(buf, (it / NUM_ACC) & 1u);
                        if (!ok) break;
                        seen = true;
                    }
                    TmemPieces pieces{tacc + ch * 32u, NP, c.kb1 == c.kb0};
                    const uint32_t block = epp->ragged == RAGGED_ROWS
                                               ? group_first_block(c.first, c.group, bs) + (col0 - c.first) / bs
                                               : c.z_out * epp->part_blocks + col0 / bs;
                    ec.chunk(c, col0, n, i, live, block, c.z_out * epp->part_blocks + c.m0 / p.bm * 4u + q, pieces, NP, side,
                             [&] { if (ch + EPI_SETS >= CHUNKS) release(buf); });
                }
                if (ok && !seen) { // fewer chunks than warps
                    ok = accumulator(buf, (it / NUM_ACC) & 1u);
                    if (ok) release(buf);
                }
            }
        } else {
            using EW = EpilogueWarp<OUT>;
            const uint32_t per_warp = (epp->bufs + epp->aux) * EPI_BUF_BYTES;
            EW ew{p, *epp, *em, tmD, p.out, lane, epi + (warp - 2u) * per_warp, ptx::smem_u32(&s_in[(warp - 2u) * 2u]),
                  s_bias, &s_abort};
            bool live_warp = true;
            for (; ok && next_work(cur, c); ++it) {
                const uint32_t buf = it % NUM_ACC;
#pragma unroll 1
                for (uint32_t hh = 0; ok && hh < static_cast<uint32_t>(NSUB); ++hh) {
                    const uint32_t bar_i  = (NSUB == 2) ? hh : buf;
                    const uint32_t parity = (NSUB == 2) ? (it & 1u) : ((it / NUM_ACC) & 1u);
                    const uint32_t colh   = c.n0 + hh * UMMA_N;
                    const uint32_t row0   = c.m0 + rank * BLOCK_M + q * 32u;
                    const uint32_t width  = FLEX ? wn : static_cast<uint32_t>(UMMA_N);
                    const uint32_t live   = (row0 < c.end && q * 32u < p.bm && colh < p.N) ? (min(width, p.N - colh) + EW::CH - 1u) / EW::CH : 0u;
                    const uint32_t mine   = live > hw ? (live - hw + EPI_SETS - 1u) / EPI_SETS : 0u; // this warp's chunks: hw, hw + EPI_SETS, ...
                    auto           col    = [&](uint32_t k) { return colh + (hw + EPI_SETS * k) * EW::CH; };
                    const uint32_t tacc   = tmem_base + ((q * 32u) << 16) + (NSUB == 2 ? hh * UMMA_N : buf * ACC_COLS);
                    float          bias_row = 0.f;
                    if (mine && live_warp) {
                        dep_wait();
                        if (epp->streamed) {
                            ew.buffers_free();
                            for (uint32_t k = 0; k < min(epp->bufs, mine); ++k) ew.request(k, row0, col(k), c.z_out);
                        }
                        bias_row = ew.row_bias(c, row0 + lane);
                    }
                    if (epp->bias && !epp->bias_on_rows) dep_wait(); // (every warp brings its share, with or without rows of its own)
                    ew.fetch_bias(c, colh, (warp - 2u) * 32u, s_bias + (waits & 1u) * BIAS_BYTES);
                    ok = accumulator(bar_i, parity);
                    if (!ok) break;
                    if (!live_warp) continue; // (it still meets the others at every accumulator)
                    if (mine == 0u) release(bar_i);
#pragma unroll 1
                    for (uint32_t k = 0; k < mine; ++k) {
                        auto read = [&] { if (k + 1u == mine) release(bar_i); };
                        if (epp->plain) {
                            ew.finish_plain(c, row0, col(k), c.end, tacc + (hw + EPI_SETS * k) * EW::CH, c.kb1 == c.kb0, read);
                            stored();
                            continue;
                        }
                        TmemPieces pieces{tacc + (hw + EPI_SETS * k) * EW::CH, EW::CH / PIECE, c.kb1 == c.kb0};
                        if (epp->streamed && k > 0u && k - 1u + epp->bufs < mine) {
                            ew.buffers_free(); // the chunk before this one left from the buffer asked for now
                            ew.request(epp->bufs - 1u, row0, col(k - 1u + epp->bufs), c.z_out);
                        }
                        live_warp = ew.finish(c, row0, col(k), col(k) - colh, c.end, bias_row, pieces, read);
                        stored();
                        if (!live_warp) break; // (a wait ran out: the abort flag ends the other roles)
                    }
                }
            }
            ew.drain();
        }
        if (warp == 2u && lane == 0) B200_TL(12);
    } else {
        // ------------------------------------------------------------------ epilogue
        const uint32_t q    = warp & 3u; // TMEM lane quarter this warp may read
        const uint32_t stg  = epi + q * 2u * EPI_BUF_BYTES;
        uint32_t       it   = 0, nstore = 0;
        bool           ok   = true;
        const uint64_t pol_d = ptx::make_l2_policy((p.l2_hints >> 4) & 3u);
        WorkCursor cur = work_begin(p, unit, krank);
        WorkCoord  c;
        if constexpr (KS) {
            // One tile per cluster: wait for this CTA's partial accumulator; the partials are
            // summed after the cluster barrier below.
            if (work_next(p, cur, unit, units, wn, tile_m, c)) {
                ok = bounded_wait(ptx::smem_u32(&s_tfull[0]), 0u, &s_abort, p.status, ST_EPI_WAIT);
                ok = __all_sync(0xffffffffu, ok);
                ptx::tc_fence_after();
                ks_c  = c;
                ks_ok = ok;
                if (warp == 2 && lane == 0) {
                    B200_TL(9);
                    B200_TL_CTA(2);
                }
            }
        } else
        for (; ok && work_next(p, cur, unit, units, wn, tile_m, c); ++it) {
            const uint32_t  buf    = it % NUM_ACC;
            const uint32_t  aphase = (it / NUM_ACC) & 1u;
            // A 512-wide tile is drained as two 256-column halves, each published (s_tfull[h])
            // and handed back (s_tempty[h]) on its own; narrower tiles have one accumulator per
            // barrier pair.
#pragma unroll 1
            for (uint32_t hh = 0; hh < static_cast<uint32_t>(NSUB); ++hh) {
            const uint32_t bar_i  = (NSUB == 2) ? hh : buf;
            const uint32_t parity = (NSUB == 2) ? (it & 1u) : aphase;
            const uint32_t colh   = hh * UMMA_N; // first column of this half within the tile
            ok = bounded_wait(ptx::smem_u32(&s_tfull[bar_i]), parity, &s_abort, p.status,
                              ST_EPI_WAIT);
            ok = __all_sync(0xffffffffu, ok); // warp-uniform: the TMEM loads below are aligned
            if (!ok) break;
            if (warp == 2 && lane == 0 && it == 0) {
                B200_TL(9);
                B200_TL_CTA(2);
            }
            ptx::tc_fence_after();
            const uint32_t row0     = c.m0 + rank * BLOCK_M + q * 32u;
            // 32-row groups at and beyond the slab height belong to the next tile (narrow staged
            // tiles may use slabs of 32, 64 or 96 rows; p.bm is 128 everywhere else).
            const bool     row_live = row0 < p.M && q * 32u < p.bm;
            const uint32_t tacc = tmem_base + ((q * 32u) << 16) + buf * ACC_COLS + colh;
            if constexpr (TR) {
                // Transposed epilogue: D(i, j) goes to out[j * M + i].  Each lane owns row i, so
                // for a fixed column j the warp writes 32 consecutive elements: coalesced stores
                // straight from registers, no staging.  Used when the caller's small dimension
                // had to become the MMA's N extent (skinny problems).
                // Rows at and beyond p.bm belong to the next slab (the MMA computed them from
                // whatever follows the slab in shared memory): never stored.
                const uint32_t i      = c.m0 + q * 32u + lane;
                const bool     i_live = (q * 32u + lane) < p.bm && i < p.M;
                dep_wait();
#pragma unroll 1
                for (int ch = 0; ch < (BN + 31) / 32; ++ch) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32(tacc + ch * 32, v);
                    ptx::tmem_ld_wait(v);
                    if (ch == (BN + 31) / 32 - 1) {
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&s_tempty[buf]));
                    }
                    if (i_live) {
                        const size_t base = (static_cast<size_t>(c.z_out) * p.N + c.n0 + ch * 32) * p.M + i;
#pragma unroll
                        for (int r = 0; r < 32; ++r) {
                            if (ch * 32 + r < BN && c.n0 + ch * 32 + r < p.N) {
                                const size_t at = base + static_cast<size_t>(r) * p.M;
                                if constexpr (OUT == OUT_F32) {
                                    static_cast<float*>(p.out)[at] = __uint_as_float(v[r]);
                                } else if constexpr (OUT == OUT_F16) {
                                    static_cast<__half*>(p.out)[at] = __float2half_rn(__uint_as_float(v[r]));
                                } else {
                                    static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(__uint_as_float(v[r]));
                                }
                            }
                        }
                    }
                }
                continue;
            }
            // Software pipeline over 128-byte column chunks: the TMEM load of chunk ch + 1 is
            // in flight while chunk ch is converted, staged and handed to the TMA store.  `O` is
            // the element kind written: the kernel's output type, or f32 for a partial tile of
            // the balanced schedule (tile-local coordinates in the workspace map `tm`).
            auto drain = [&](auto out_tag, const CUtensorMap* tm, bool tile_local) {
            constexpr int O    = decltype(out_tag)::value;
            constexpr int O_CH = (O == OUT_F32) ? 32 : 64; // output columns per 128-byte chunk
            uint32_t       n0[32], n1[32]; // raw accumulator words of the chunk in flight
            ptx::tmem_ld_32x32(tacc, n0);
            if constexpr (O != OUT_F32) ptx::tmem_ld_32x32(tacc + 32u, n1);
            const int NCH_H = FLEX ? static_cast<int>(wn) / O_CH : (BN < O_CH ? 1 : BN / O_CH) / NSUB; // chunks per half
#pragma unroll 1
            for (int ch = 0; ch < NCH_H; ++ch) {
                uint32_t v[32];
                ptx::tmem_ld_wait(n0);
                if constexpr (O == OUT_F32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = n0[j];
                } else {
                    ptx::tmem_ld_wait(n1);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v[j]      = pack2<O>(n0[2 * j], n0[2 * j + 1]);
                        v[16 + j] = pack2<O>(n1[2 * j], n1[2 * j + 1]);
                    }
                }
                if (ch + 1 < NCH_H) {
                    ptx::tmem_ld_32x32(tacc + (ch + 1) * O_CH, n0);
                    if constexpr (O != OUT_F32) ptx::tmem_ld_32x32(tacc + (ch + 1) * O_CH + 32u, n1);
                }
                if (ch == NCH_H - 1) {
                    // Accumulator (half) fully read: hand it back to the MMA issuer (rank 0).
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (CL == 2) ptx::mbar_arrive_cluster(ptx::smem_u32(&s_tempty[bar_i]), 0);
                        else ptx::mbar_arrive(ptx::smem_u32(&s_tempty[bar_i]));
                    }
                }
                const uint32_t col0 = c.n0 + colh + ch * O_CH;
                if (row_live && col0 < p.N) {
                    const uint32_t sbuf = stg + (nstore & 1u) * EPI_BUF_BYTES;
                    // The store that last used this buffer (two stores ago) must have read it.
                    if (lane == 0) ptx::tma_store_wait_read<1>();
                    __syncwarp();
                    const uint32_t rowaddr = sbuf + lane * 128u;
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        st_shared_v4(rowaddr + ((j ^ (lane & 7u)) << 4), v[4 * j], v[4 * j + 1],
                                     v[4 * j + 2], v[4 * j + 3]);
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        dep_wait();
                        if constexpr (GATHER) {
                            // The tile goes to every copy of the full matrix (this GPU's and its
                            // peers', over NVLink) at the slab's offset: the all-gather of the
                            // output happens tile by tile under the main loop of the next tile.
                            for (uint32_t d = 0; d < p.ndst; ++d)
                                ptx::tma_store_3d(&tmDs[d], sbuf, col0 + p.dst_col0, row0 + p.dst_row0, c.z_out, pol_d);
                        } else if (tile_local) {
                            ptx::tma_store_3d(tm, sbuf, col0 - c.n0, row0 - c.m0, c.z_out, pol_d);
                        } else {
                            ptx::tma_store_3d(tm, sbuf, col0, row0, c.z_out, pol_d);
                        }
                        ptx::tma_store_commit();
                        if (warp == 2) {
                            if (nstore == 0) B200_TL(10);
                            B200_TL(11);
                        }
                    }
                    ++nstore;
                }
            }
            }; // drain
            if constexpr (!GATHER && NSUB == 1 && !TR) {
                // balanced schedule: partial segments go to the workspace as f32, whole tiles to C
                if (c.partial) drain(std::integral_constant<int, OUT_F32>{}, &tmW, true);
                else drain(std::integral_constant<int, OUT>{}, &tmD, false);
            } else {
                drain(std::integral_constant<int, OUT>{}, &tmD, false);
            }
            } // halves
        }
        // The staging buffers may go away once the stores have READ them; the writes themselves
        // are complete when the grid is (and a dependent grid waits for exactly that).
        if (lane == 0) ptx::tma_store_wait_read<0>();
        if (warp == 2 && lane == 0) B200_TL(12);
    }

    if constexpr (KS) {
        // ------------------------------------------------------ sum of the cluster's K partitions
        // Every CTA of the cluster holds an f32 partial of the same tile in TMEM.  The tile's
        // 128-byte output chunks are dealt round-robin to the CTAs (chunk ch belongs to rank
        // ch % split_k); each CTA sends the chunks it does not own to their owners' shared memory
        // (the operand ring, free once every CTA's MMAs have retired: first barrier), and after the
        // second barrier adds the partials of its own chunks in partition order - whichever CTA
        // owns a chunk, the sum is ((p0 + p1) + p2) + ... - converts and stores them to C.  No
        // workspace in global memory and no second kernel.  All threads of the cluster pass both
        // barriers whatever happened before (a role that gave up a bounded wait included).
        // (the transposed epilogue stores element by element: its chunks are 32 f32 columns)
        constexpr int      O_CH  = (TR || OUT == OUT_F32) ? 32 : 64; // output columns per chunk
        constexpr int      NCH   = TR ? (BN + 31) / 32 : BN / O_CH; // (a 16-column slab is one chunk, half of it unused)
        constexpr uint32_t ROW_B = O_CH * 4u;                  // bytes of one row of an f32 chunk
        constexpr uint32_t WSLOT = 32u * ROW_B;                // one warp's 32 rows of a chunk
        const uint32_t ks   = p.split_k;
        const uint32_t q    = warp & 3u;
        const uint32_t tacc = tmem_base + ((q * 32u) << 16);
        const uint32_t hw   = EP && warp >= 2u ? (warp - 2u) >> 2 : 0u; // EP: two warps per quarter, a rank's chunks dealt alternately
        __syncwarp();
        if (warp == 2 && lane == 0) B200_TL(16);
        ptx::cluster_arrive();
        ptx::cluster_wait();
        if (warp == 2 && lane == 0) B200_TL(17);
        if (warp >= 2 && ks_ok) {
#pragma unroll 1
            for (uint32_t ch = 0; ch < static_cast<uint32_t>(NCH); ++ch) {
                const uint32_t owner = ch % ks;
                if (owner == krank) continue;
                if (EP && (ch / ks) % EPI_SETS != hw) continue;
                // (within a warp's slot the 16-byte units are laid out [unit][lane]: every store and
                // load instruction of the warp covers 512 contiguous bytes)
                const uint32_t local  = ring + (((ch / ks) * ks + krank) * 4u + q) * WSLOT + lane * 16u;
                const uint32_t remote = ptx::mapa_u32(local, owner);
#pragma unroll
                for (uint32_t h = 0; h < static_cast<uint32_t>(O_CH / 32); ++h) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32(tacc + ch * O_CH + h * 32u, v);
                    ptx::tmem_ld_wait(v);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j)
                        ptx::st_cluster_v4(remote + (h * 8u + j) * 512u, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
            }
        }
        __syncwarp();
        if (warp == 2 && lane == 0) B200_TL(18);
        ptx::cluster_arrive();
        ptx::cluster_wait();
        if (warp == 2 && lane == 0) B200_TL(19);
        if (warp >= 2 && ks_ok) {
            const uint32_t stg      = epi + q * 2u * EPI_BUF_BYTES;
            const uint32_t row0     = ks_c.m0 + q * 32u;
            const bool     row_live = row0 < p.M;
            uint32_t       nstore   = 0;
            [[maybe_unused]] const uint32_t per_warp = EP ? (epp->bufs + epp->aux) * EPI_BUF_BYTES : 0u;
            auto make_ew = [&]() {
                if constexpr (EP && !TR)
                    return EpilogueWarp<OUT>{p, *epp, *em, tmD, p.out, lane, epi + (warp - 2u) * per_warp,
                                             ptx::smem_u32(&s_in[(warp - 2u) * 2u]), s_bias, &s_abort};
                else return 0;
            };
            [[maybe_unused]] auto ew = make_ew();
#pragma unroll 1
            for (uint32_t ch = krank + (EP ? hw * ks : 0u); ch < static_cast<uint32_t>(NCH); ch += (EP ? EPI_SETS : 1u) * ks) {
                if constexpr (EP) {
                    ClusterPieces pieces{tacc + ch * O_CH, ring + ((ch / ks) * ks * 4u + q) * WSLOT + lane * 16u, 4u * WSLOT, ks, krank};
                    dep_wait();
                    if constexpr (TR) {
                        const EpilogueColumns<OUT> ec{p, *epp, lane};
                        const uint32_t i    = ks_c.m0 + q * 32u + lane;
                        const bool     live = (q * 32u + lane) < p.bm && i < p.M;
                        const uint32_t col0 = ks_c.n0 + ch * 32u;
                        const uint32_t bs   = BN < 32 ? BN : 32;
                        const uint32_t n    = col0 < p.N ? min(min(32u, BN - ch * 32u), p.N - col0) : 0u;
                        float          side[PIECE];
                        if (epp->streamed) ec.load_side(ks_c, col0, min(n, static_cast<uint32_t>(PIECE)), i, live, side);
                        ec.chunk(ks_c, col0, n, i, live, ks_c.z_out * epp->part_blocks + col0 / bs,
                                 ks_c.z_out * epp->part_blocks + ks_c.m0 / p.bm * 4u + q, pieces, bs / PIECE, side, [] {});
                    } else {
                        const uint32_t col0 = ks_c.n0 + ch * O_CH;
                        if (row_live && col0 < p.N) {
                            if (epp->streamed) {
                                ew.buffers_free();
                                ew.request(0u, row0, col0, ks_c.z_out);
                            }
                            if (!ew.finish(ks_c, row0, col0, ch * O_CH, p.M, ew.row_bias(ks_c, row0 + lane), pieces, [] {})) break;
                        }
                    }
                } else {
                uint32_t own[O_CH];
                float    acc[O_CH];
#pragma unroll
                for (uint32_t h = 0; h < static_cast<uint32_t>(O_CH / 32); ++h) {
                    uint32_t t[32];
                    ptx::tmem_ld_32x32(tacc + ch * O_CH + h * 32u, t);
                    ptx::tmem_ld_wait(t);
#pragma unroll
                    for (int j = 0; j < 32; ++j) own[h * 32 + j] = t[j];
                }
#pragma unroll 1
                for (uint32_t s = 0; s < ks; ++s) {
                    if (s == krank) {
#pragma unroll
                        for (int j = 0; j < O_CH; ++j)
                            acc[j] = (s == 0u) ? __uint_as_float(own[j]) : acc[j] + __uint_as_float(own[j]);
                    } else {
                        const uint32_t src = ring + (((ch / ks) * ks + s) * 4u + q) * WSLOT + lane * 16u;
#pragma unroll
                        for (uint32_t h = 0; h < static_cast<uint32_t>(O_CH / 32); ++h) {
#pragma unroll
                            for (uint32_t j = 0; j < 8; ++j) {
                                uint32_t x0, x1, x2, x3;
                                ptx::ld_shared_v4(src + (h * 8u + j) * 512u, x0, x1, x2, x3);
                                const int at = h * 32 + 4 * j;
                                acc[at]     = (s == 0u) ? __uint_as_float(x0) : acc[at] + __uint_as_float(x0);
                                acc[at + 1] = (s == 0u) ? __uint_as_float(x1) : acc[at + 1] + __uint_as_float(x1);
                                acc[at + 2] = (s == 0u) ? __uint_as_float(x2) : acc[at + 2] + __uint_as_float(x2);
                                acc[at + 3] = (s == 0u) ? __uint_as_float(x3) : acc[at + 3] + __uint_as_float(x3);
                            }
                        }
                    }
                }
                if constexpr (TR) {
                    // D(i, j) goes to out[j * M + i]: for a fixed column the warp writes 32
                    // consecutive elements (see the transposed epilogue above).
                    const uint32_t i      = ks_c.m0 + q * 32u + lane;
                    const bool     i_live = (q * 32u + lane) < p.bm && i < p.M;
                    dep_wait();
                    if (i_live) {
                        const size_t base = (static_cast<size_t>(ks_c.z_out) * p.N + ks_c.n0 + ch * 32u) * p.M + i;
#pragma unroll
                        for (int r = 0; r < 32; ++r) {
                            if (ks_c.n0 + ch * 32u + r < p.N) {
                                const size_t at = base + static_cast<size_t>(r) * p.M;
                                if constexpr (OUT == OUT_F32) static_cast<float*>(p.out)[at] = acc[r];
                                else if constexpr (OUT == OUT_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(acc[r]);
                                else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(acc[r]);
                            }
                        }
                    }
                } else {
                uint32_t v[32];
                if constexpr (OUT == OUT_F32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(acc[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = pack2<OUT>(__float_as_uint(acc[2 * j]), __float_as_uint(acc[2 * j + 1]));
                }
                const uint32_t col0 = ks_c.n0 + ch * O_CH;
                if (row_live && col0 < p.N) {
                    const uint32_t sbuf = stg + (nstore & 1u) * EPI_BUF_BYTES;
                    if (lane == 0) ptx::tma_store_wait_read<1>();
                    __syncwarp();
                    const uint32_t rowaddr = sbuf + lane * 128u;
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j)
                        st_shared_v4(rowaddr + ((j ^ (lane & 7u)) << 4), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        dep_wait();
                        ptx::tma_store_3d(&tmD, sbuf, col0, row0, ks_c.z_out, ptx::make_l2_policy((p.l2_hints >> 4) & 3u));
                        ptx::tma_store_commit();
                    }
                    ++nstore;
                }
                } // staged store
                } // without an epilogue
            }
            if (warp == 2 && lane == 0) B200_TL(20);
            if constexpr (EP && !TR) ew.drain();
            if (lane == 0) ptx::tma_store_wait_read<0>();
            if (warp == 2 && lane == 0) B200_TL(21);
        }
    }

    // ---------------------------------------------------------------------- tail
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (CL == 2) { // neither CTA may leave while its peer can still touch it
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (threadIdx.x == 0) B200_TL(13);
    if (threadIdx.x == 64) B200_TL_CTA(1);
    if (warp == 1) {
        ptx::tc_fence_after();
        __syncwarp();
        ptx::tmem_dealloc<CL>(tmem_base, TMEM_COLS);
        if (lane == 0) B200_TL(14);
    }
}

template <int BN, int OUT, int CL, bool TR = false>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    gemm_umma_kernel(const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmD,
                     const __grid_constant__ CUtensorMap tmW, const GemmParams p)
{
    // tmW: the balanced schedule's workspace of f32 partial tiles (any valid map otherwise)
    gemm_umma_body<BN, OUT, CL, TR, false>(tmA, tmB, &tmD, tmW, p);
}

// The same GEMM with the all-gather of its output fused into the epilogue: this GPU computes a
// slab of a larger matrix and stores every tile of it into p.ndst copies of that matrix (its own
// and, through peer mappings, the other GPUs').  Plain TMA stores to peer memory: no loads from
// a peer, no multicast, and no wait on another GPU anywhere in the kernel.
template <int BN, int OUT, int CL>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    gemm_umma_gather_kernel(const __grid_constant__ CUtensorMap tmA,
                            const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ GatherMaps dst, const GemmParams p)
{
    gemm_umma_body<BN, OUT, CL, false, true>(tmA, tmB, dst.m, dst.m[0], p);
}

// The same GEMM with a tile's K partitions spread over the CTAs of a cluster (cluster size =
// p.split_k, one tile per cluster) and summed through distributed shared memory.
template <int BN, int OUT, bool TR = false>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    gemm_umma_ksplit_kernel(const __grid_constant__ CUtensorMap tmA,
                            const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ CUtensorMap tmD, const GemmParams p)
{
    gemm_umma_body<BN, OUT, 1, TR, false, true>(tmA, tmB, &tmD, tmD, p);
}

// The GEMM with an epilogue, dense or grouped, and its form with cluster K partitions.
template <int BN, int OUT, int CL, bool TR = false>
__global__ void __launch_bounds__(EPI_THREADS, 1)
    gemm_epilogue_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmD, const __grid_constant__ EpilogueMaps em,
                         const GemmParams p, const EpilogueParams ep)
{
    gemm_umma_body<BN, OUT, CL, TR, false, false, true>(tmA, tmB, &tmD, tmD, p, &em, &ep);
}

template <int BN, int OUT, bool TR = false>
__global__ void __launch_bounds__(EPI_THREADS, 1)
    gemm_epilogue_ksplit_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                                const __grid_constant__ CUtensorMap tmD, const __grid_constant__ EpilogueMaps em,
                                const GemmParams p, const EpilogueParams ep)
{
    gemm_umma_body<BN, OUT, 1, TR, false, true, true>(tmA, tmB, &tmD, tmD, p, &em, &ep);
}

// A copy of `lines` lines of `length` 16-bit elements with every line padded to `pitch` elements (a
// multiple of 8) of zeros, for operands whose lines do not start on 16-byte boundaries: TMA
// addresses the copy.  HBM-bound: (2 length + 2 pitch) bytes per line.
static __global__ void __launch_bounds__(256)
    pad_lines_kernel(const uint16_t* src, uint4* dst, uint64_t units, uint32_t length, FastDiv per_line)
{
    for (uint64_t u = blockIdx.x * 256ull + threadIdx.x; u < units; u += gridDim.x * 256ull) {
        uint64_t line;
        uint32_t at;
        if (units < 0x80000000ull) {
            line = fast_div(static_cast<uint32_t>(u), per_line);
            at   = static_cast<uint32_t>(u) - static_cast<uint32_t>(line) * per_line.d;
        } else {
            line = u / per_line.d;
            at   = static_cast<uint32_t>(u - line * per_line.d);
        }
        const uint16_t* from = src + line * length + at * 8u;
        uint32_t        w[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t e  = at * 8u + 2u * k;
            const uint32_t lo = e < length ? from[2 * k] : 0u, hi = e + 1u < length ? from[2 * k + 1] : 0u;
            w[k]              = lo | (hi << 16);
        }
        dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Maps of a ragged-K product: group e's copies of the two operands' maps, with the row extent
// ending at the group's end, so that the K loop's last box is zero-filled there instead of
// reading the next group's rows.  One warp per group.
static __global__ void __launch_bounds__(32)
    ragged_maps_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       CUtensorMap* __restrict__ maps, const int32_t* offsets, uint32_t rows)
{
    const uint32_t e = blockIdx.x, lane = threadIdx.x;
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();
    uint32_t lo, hi;
    group_rows(offsets, e, rows, lo, hi);
    if (lane < 16u) {
        const uint64_t* src = reinterpret_cast<const uint64_t*>(&tmA);
        const uint64_t* srb = reinterpret_cast<const uint64_t*>(&tmB);
        uint64_t*       dst = reinterpret_cast<uint64_t*>(maps + 2u * e);
        dst[lane]           = src[lane];
        dst[16u + lane]     = srb[lane];
    }
    __syncwarp();
    if (lane < 2u) {
        ptx::tensormap_set_dim1(maps + 2u * e + lane, max(hi, 1u)); // (an extent may not be 0; such a group loads nothing)
        ptx::fence_tensormap_release();
    }
}

// ---------------------------------------------------------------------------------------------
// Split-K reduction: out[z][i] = convert(sum_s ws[z][s][i]), s ascending (deterministic).
// `ws` holds batch * split_k partial matrices of `mn` f32 elements each.
// ---------------------------------------------------------------------------------------------
template <int OUT>
__global__ void __launch_bounds__(256)
    splitk_reduce_kernel(const float* __restrict__ ws, void* __restrict__ out, uint64_t mn,
                         uint32_t split_k, uint32_t batch)
{
    const uint64_t total4 = (mn * batch) >> 2; // mn is a multiple of 4
    const uint64_t mn4    = mn >> 2;
    ptx::grid_dep_wait(); // the partials are complete once the GEMM grid before this one has finished
    ptx::grid_dep_launch();
    for (uint64_t i = blockIdx.x * static_cast<uint64_t>(blockDim.x) + threadIdx.x; i < total4;
         i += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
        const uint64_t z   = i / mn4;
        const uint64_t e   = i - z * mn4;
        const float4*  src = reinterpret_cast<const float4*>(ws) + z * split_k * mn4 + e;
        float4         acc = __ldg(src);
        for (uint32_t s = 1; s < split_k; ++s) {
            const float4 t = __ldg(src + s * mn4);
            acc.x += t.x;
            acc.y += t.y;
            acc.z += t.z;
            acc.w += t.w;
        }
        if constexpr (OUT == OUT_F32) {
            reinterpret_cast<float4*>(out)[i] = acc;
        } else if constexpr (OUT == OUT_F16) {
            const __half2 a = __floats2half2_rn(acc.x, acc.y);
            const __half2 b = __floats2half2_rn(acc.z, acc.w);
            uint2         u;
            u.x = *reinterpret_cast<const uint32_t*>(&a);
            u.y = *reinterpret_cast<const uint32_t*>(&b);
            reinterpret_cast<uint2*>(out)[i] = u;
        } else {
            const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x, acc.y);
            const __nv_bfloat162 b = __floats2bfloat162_rn(acc.z, acc.w);
            uint2                u;
            u.x = *reinterpret_cast<const uint32_t*>(&a);
            u.y = *reinterpret_cast<const uint32_t*>(&b);
            reinterpret_cast<uint2*>(out)[i] = u;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Fix-up pass of the balanced (stream-K) schedule: for every tile that a run boundary cuts,
// out(tile) = convert(sum of the tile's partial tiles), partials added in K order (ascending
// worker), so the result does not depend on timing.  Tiles no boundary cuts were written to C
// by the GEMM kernel itself and are not touched.
//
// Job j (1 <= j < workers) belongs to the boundary between runs j - 1 and j.  The boundary cuts
// a tile unless it falls on a tile's first K step; a tile cut by several boundaries is handled
// by the job of the first of them.  The tile's contributors are the workers w0 .. w1 whose runs
// hold its first and last K step; worker w's partial sits in slot 2w if its run starts inside
// the tile, in slot 2w + 1 if its run came in through the tile's first K step (see WorkCursor).
// `ws` holds one dense tile_m x tile_n f32 tile per slot.  N is a multiple of 4, so a float4
// never straddles the matrix edge.  L2/HBM-bound: (parts x 4 + sizeof(out)) bytes per element
// of a cut tile; blockIdx.y = job, blockIdx.x strides over the tile's float4s.
// ---------------------------------------------------------------------------------------------
template <int OUT>
__global__ void __launch_bounds__(256)
    streamk_reduce_kernel(const float* __restrict__ ws, void* __restrict__ out, const GemmParams p, uint32_t tile_m,
                          uint32_t tile_n)
{
    ptx::grid_dep_wait(); // the partials are complete once the GEMM grid before this one has finished
    ptx::grid_dep_launch();
    const uint32_t j        = blockIdx.y + 1u;
    const uint32_t upt      = p.units_per_tile;
    const uint32_t boundary = run_start(p, j);
    const uint32_t tile     = boundary / upt; // over batch x tiles
    const uint32_t tile_beg = tile * upt;
    if (boundary == tile_beg) return;                             // the cut falls between two tiles
    if (j > 1u && run_start(p, j - 1u) > tile_beg) return;        // an earlier boundary owns this tile
    // workers whose runs hold the tile's first and last K step
    const uint64_t x0 = tile_beg, x1 = x0 + upt - 1u;
    const uint32_t w0 = static_cast<uint32_t>(((x0 + 1u) * p.workers + p.total_units - 1u) / p.total_units) - 1u;
    const uint32_t w1 = static_cast<uint32_t>(((x1 + 1u) * p.workers + p.total_units - 1u) / p.total_units) - 1u;
    const uint32_t tiles    = p.m_tiles * p.n_tiles;
    const uint32_t row4     = tile_n / 4u; // float4 per tile row
    const uint32_t tile_sz4 = tile_m * row4;
    uint32_t       m_idx, n_idx;
    tile_coords(p, tile % tiles, m_idx, n_idx);
    const uint32_t z    = tile / tiles;
    const float4*  ws4  = reinterpret_cast<const float4*>(ws);
    // the first contributor's run holds the tile's first K step: its partial is its run's last segment
    const uint32_t slot0 = 2u * w0 + 1u;
    for (uint32_t e = blockIdx.x * blockDim.x + threadIdx.x; e < tile_sz4; e += gridDim.x * blockDim.x) {
        const uint32_t rr = e / row4, c4 = e - rr * row4;
        const uint32_t row = m_idx * tile_m + rr, col = n_idx * tile_n + c4 * 4u;
        if (row >= p.M || col >= p.N) continue;
        float4 acc = __ldg(ws4 + static_cast<uint64_t>(slot0) * tile_sz4 + e);
        for (uint32_t w = w0 + 1u; w <= w1; ++w) { // these runs start inside the tile: slot 2w
            const float4 t = __ldg(ws4 + static_cast<uint64_t>(2u * w) * tile_sz4 + e);
            acc.x += t.x;
            acc.y += t.y;
            acc.z += t.z;
            acc.w += t.w;
        }
        const uint64_t at = (static_cast<uint64_t>(z) * p.M + row) * p.N + col; // element index; col % 4 == 0
        if constexpr (OUT == OUT_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = acc;
        } else if constexpr (OUT == OUT_F16) {
            const __half2 a = __floats2half2_rn(acc.x, acc.y);
            const __half2 b = __floats2half2_rn(acc.z, acc.w);
            uint2         u;
            u.x = *reinterpret_cast<const uint32_t*>(&a);
            u.y = *reinterpret_cast<const uint32_t*>(&b);
            *reinterpret_cast<uint2*>(static_cast<__half*>(out) + at) = u;
        } else {
            const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x, acc.y);
            const __nv_bfloat162 b = __floats2bfloat162_rn(acc.z, acc.w);
            uint2                u;
            u.x = *reinterpret_cast<const uint32_t*>(&a);
            u.y = *reinterpret_cast<const uint32_t*>(&b);
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at) = u;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// CUDA-core GEMM with arbitrary element strides, f32 accumulation in ascending k.  Only used
// for shapes whose contiguous extents are not multiples of 16 bytes (TMA cannot address
// them); correctness path, not a performance path.
// ---------------------------------------------------------------------------------------------
template <class TIn, class TOut>
__global__ void __launch_bounds__(256)
    gemm_generic_kernel(TOut* __restrict__ C, const TIn* __restrict__ A,
                        const TIn* __restrict__ B, uint32_t M, uint32_t N, uint32_t K,
                        uint64_t a_sm, uint64_t a_sk, uint64_t b_sk, uint64_t b_sn, uint64_t c_sm,
                        uint64_t c_sn, uint64_t a_sb, uint64_t b_sb, uint64_t c_sb)
{
    __shared__ float sA[16][17];
    __shared__ float sB[16][17];
    const uint32_t   tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    const uint32_t   i = blockIdx.y * 16u + ty, j = blockIdx.x * 16u + tx;
    const TIn*       Ab  = A + blockIdx.z * a_sb;
    const TIn*       Bb  = B + blockIdx.z * b_sb;
    float            acc = 0.f;
    for (uint32_t k0 = 0; k0 < K; k0 += 16u) {
        const uint32_t ka = k0 + tx, kb = k0 + ty;
        sA[ty][tx] = (i < M && ka < K) ? static_cast<float>(Ab[i * a_sm + ka * a_sk]) : 0.f;
        sB[ty][tx] = (kb < K && j < N) ? static_cast<float>(Bb[kb * b_sk + j * b_sn]) : 0.f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) acc += sA[ty][k] * sB[k][tx];
        __syncthreads();
    }
    if (i < M && j < N) C[blockIdx.z * c_sb + i * c_sm + j * c_sn] = static_cast<TOut>(acc);
}

} // namespace b200
