// Dense non-causal attention forward for gfx950 (MI355X), bf16 in / bf16 out,
// fp32 log-sum-exp. Semantics follow the FlashAttention-4 call made by the
// reference adapter (src/h3_flash/runtime/attention/dense_fa4.py:74-80,145):
// O = softmax(scale * Q K^T) V over the full key range of each (batch, head),
// or of each packed segment when cu_seqlens are given.
//
// The tile and its pipeline are described in attn_tile.h.
#include <atomic>
#include <type_traits>

#include "attn_tile.h"
#include "common.h"
#include "kernels.h"

// Workspace of h3a_attn_fwd_noalloc: the partial results (O, fp32 LSE) of the tail's
// key-range pieces and the tail's counter, for callers that cannot allocate.
// Every GPU the library runs on holds its own copy until the process ends.
// Host code never passes `scratch` itself (on the host it names a shadow
// variable, not device memory): attn_static_scratch looks up this device's
// copy with hipGetSymbolAddress and kernels take that address.
static __device__ __align__(256) char scratch[h3a::kStaticScratchBytes];

namespace h3a {
namespace {

constexpr int kPersistMaxQTiles = 16;  // longest segment of a persistent launch: 4,096 rows
// Fewest key tiles in such a piece: each piece pays a pipeline fill and
// drain and a partial result, which short pieces do not recover (8 x 8,192-row
// segments at 5 heads cut into pieces of 32 key tiles ran 5% slower).
constexpr int kQueueMinKeyTiles = 48;
// Times in a launch's last round (plan_attn_last_round), in us: the fixed part of a
// tile or piece, and the launches that pieces add. At most kMaxPieces pieces.
constexpr double kTileUs = 9.7, kPiecesUs = 14.0;
constexpr int kMaxPieces = 8;

// The unit of rows [m0, m0 + 32) of head h of batch (or packed segment) grp.
template <typename Params>
__device__ __forceinline__ void attn_unit_at(Params& p, int grp, int h, int m0) {
    int b = grp, q0 = 0, k0 = 0, sq = p.seqlen_q, sk = p.seqlen_k;
    if (p.cu_q != nullptr) {
        b = 0;
        q0 = min(max(p.cu_q[grp], 0), p.seqlen_q);
        sq = min(max(p.cu_q[grp + 1], q0), p.seqlen_q) - q0;
        k0 = min(max(p.cu_k[grp], 0), p.seqlen_k);
        sk = min(max(p.cu_k[grp + 1], k0), p.seqlen_k) - k0;
    }
    if (m0 >= sq) return;  // the whole workgroup: past this segment
    attn_unit(p, UnitView{(const char*)p.q + 2 * (b * p.q_sb + h * p.q_sh) + (int64_t)(q0 + m0) * p.q_rs,
                          (const char*)p.k + 2 * (b * p.k_sb + h * p.k_sh) + (int64_t)k0 * p.k_rs,
                          (const char*)p.v + 2 * (b * p.v_sb + h * p.v_sh) + (int64_t)k0 * p.v_rs,
                          (char*)p.o + 2 * (b * p.o_sb + h * p.o_sh) + (int64_t)(q0 + m0) * p.o_rs,
                          p.lse == nullptr ? nullptr : p.lse + b * p.lse_sb + h * p.lse_sh + q0 + m0, sq - m0, sk});
}

// A launch of units alone, contiguous per XCD (a head's units share its K/V in
// that XCD's L2). Dense: n_units per (batch, head). Packed: the units of the
// segments one after another, a segment's heads outermost; which segment a
// workgroup's unit lies in is found from the offsets (64 segments at a time, a
// lane each), so no workgroup goes to the rows that shorter segments lack (a
// grid of n_units per segment: 14 segments of 1 to 486 rows, 8 heads, 51 us;
// this one 36). Workgroups past the last unit end at once.
__global__ __launch_bounds__(kThreads, 2) void attn_short_kernel(AttnParams p) {
    const int nb = gridDim.x, bid = blockIdx.x;
    const int xcd = bid & 7, per = nb >> 3, rem = nb & 7;
    int unit = xcd * per + min(xcd, rem) + (bid >> 3);
    if (p.cu_q == nullptr) {
        const int rest = unit / p.n_units;
        attn_unit_at(p, rest / p.heads, rest % p.heads, unit % p.n_units * kUnitRows);
        return;
    }
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < p.n_groups; s0 += 64) {
        const int s = s0 + lane;
        int n = 0;
        if (s < p.n_groups) {
            const int q0 = min(max(p.cu_q[s], 0), p.seqlen_q), q1 = min(max(p.cu_q[s + 1], q0), p.seqlen_q);
            n = min((q1 - q0 + kUnitRows - 1) / kUnitRows, p.n_units);
        }
        int incl = n * p.heads;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(incl, off, 64);
            if (lane >= off) incl += up;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl > unit);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            const int units = __builtin_amdgcn_readlane(n, at);
            unit -= __builtin_amdgcn_readlane(incl, at) - units * p.heads;
            attn_unit_at(p, s0 + at, unit / units, unit % units * kUnitRows);
            return;
        }
        unit -= __builtin_amdgcn_readlane(incl, 63);
    }
}

// The dynamic tail: the last round's tiles are cut into key-range pieces
// that the workgroups after the whole tiles take from a counter in the
// workspace as they free up, so CUs that ran their whole tiles faster (XCD
// clocks differ) take more of the tail.
template <bool kWide, bool kVT, bool kPartF32 = false>
__global__ __launch_bounds__(kThreads, 2) void attn_fwd_kernel(AttnParams p) {
    __shared__ int queue_head;
    // Workgroups are dispatched round-robin over the 8 XCDs, workgroup i to
    // XCD i % 8 as its (i / 8)-th. Dense grids are renumbered so that each
    // XCD runs one contiguous range of tiles: its 32 resident workgroups are
    // then consecutive query tiles of one head and stream that head's K/V
    // through the XCD's L2 once per round (0.98 GB of HBM reads per launch at
    // B=1 H=5 S=49,920; 1.70 GB in dispatch order, at the same speed). A
    // static split (fewer tiles than CUs, n_full == 0) gives every workgroup
    // one piece, each XCD a contiguous range of them.
    // Packed varlen launches with a work list (vplan) run the list's whole
    // rounds in dispatch order and take the last round's pieces from a
    // counter. Without a list they keep dispatch order too (tile i is
    // workgroup i): tiles past a short segment's end exit at once, and in
    // dispatch order they spread over all XCDs (contiguous ranges gave a few
    // XCDs nearly only empty tiles: the 49,920 + 1,296 two-segment batch ran
    // at half speed).
    const int bid = blockIdx.x;
    // Dense launches whose last query tile would hold at most 32 rows run
    // those as units, one per (batch, head), on the last rag_blocks workgroups:
    // a tile for them keeps a CU as long as one or two rows of tiles do (40
    // heads of 1,560 x 1,560, 240 whole tiles on 256 CUs: 66.9 -> 53.8 us).
    const int n_blocks = (int)gridDim.x - p.rag_blocks;
    if constexpr (!kWide) {
        if (bid >= n_blocks) {
            for (int u = bid - n_blocks; u < p.heads * p.n_groups; u += p.rag_blocks) {
                attn_unit_at(p, u / p.heads, u % p.heads, p.n_qtiles * kBM);
                __syncthreads();  // the merge has read the buffers that the next unit fills
            }
            return;
        }
    }
    // First work item of this wave (wide forms: read once, kept as a scalar).
    const int wave_first = kWide ? __builtin_amdgcn_readfirstlane((int)threadIdx.x) & ~63 : 0;
    int tile = bid, chunk = -1, chunks = 1, slot = -1;
    const bool planned = p.vplan != nullptr;
    // With a tail queue, the workgroups after the whole tiles take the pieces
    // of the last round's tiles from a counter, one at a time.
    const bool queued = planned ? bid >= p.ub_tiles : p.queue != nullptr && bid >= p.n_full;
    if (planned && !queued) {
        // Dispatch order over the list: its tiles differ in length (longest
        // first), and round-robin over the XCDs gives every XCD an even share
        // of each length (XCD-contiguous ranges gave XCD 0 all the longest).
        if (bid >= p.vplan[kPlanFull]) return;
        tile = __builtin_amdgcn_readfirstlane(p.vlist[bid]);  // uniform: the addressing is scalar
    } else if (p.cu_q == nullptr && !queued) {
        const int nb = p.queue != nullptr ? p.n_full : n_blocks;
        const int xcd = bid & 7, local = bid >> 3, per = nb >> 3, rem = nb & 7;
        const int start = xcd * per + min(xcd, rem);  // first tile of this XCD's share
        tile = start + local;
        if (p.split_n != 0) {
            const int full_per = p.n_full >> 3;  // n_full: 0, or whole rounds of CUs (a multiple of 8)
            if (local < full_per) {
                tile = xcd * full_per + local;
            } else {
                slot = start - xcd * full_per + (local - full_per);
                tile = p.n_full + slot % p.split_tiles;
                chunk = slot / p.split_tiles;
                chunks = p.split_n;
            }
        }
    }
    // Two call sites: the whole tiles keep a straight-line copy of the tile
    // code (a single call inside the loop below changed its register
    // allocation and made it 1-2% slower).
    if (!queued) {
        attn_tile<kWide, kVT, false, kPartF32>(p, tile, chunk, chunks, slot, false, nullptr, false, -1, nullptr, nullptr, wave_first);
        return;
    }
    int* const counter = planned ? (int*)p.vplan + kPlanQueue : p.queue;
    // The wide forms find the first work item from wave_first and the lane,
    // so no VGPR holds the id across the loop.
    const bool leader = kWide ? wave_first + lane_from_hw() == 0 : threadIdx.x == 0;
    for (;;) {
        if (leader) queue_head = atomicAdd(counter, 1);
        __syncthreads();  // also: every wave is done with the previous piece's LDS
        const int piece = __builtin_amdgcn_readfirstlane(queue_head);  // uniform: keep it scalar
        __syncthreads();  // every wave has read queue_head before it is written again
        if (planned) {
            if (piece >= p.vplan[kPlanPieces]) return;
            // pieces[i] = (list position, chunk | chunks << 2 | (merge slot + 1) << 5)
            const int pos = __builtin_amdgcn_readfirstlane(p.vpieces[2 * piece]);
            const int code = __builtin_amdgcn_readfirstlane(p.vpieces[2 * piece + 1]);
            const int merge_slot = (code >> 5) - 1;
            tile = __builtin_amdgcn_readfirstlane(p.vlist[pos]);
            chunk = code & 3;
            chunks = (code >> 2) & 7;
            slot = merge_slot >= 0 ? merge_slot * kQueuePieces + chunk : -1;
        } else {
            if ((unsigned)piece >= (unsigned)(p.split_n * p.split_tiles)) return;
            tile = p.n_full + piece % p.split_tiles;
            chunk = piece / p.split_tiles;  // chunk-major: every tile's first pieces first
            chunks = p.split_n;
            slot = piece;
        }
        // The launch arguments are read afresh for each piece (an opaque zero
        // offset keeps the compiler from hoisting the loads), from the
        // kernel-argument segment through the scalar cache, rather than held
        // in scalar registers across the loop: the piece's own addressing
        // needs those registers (spills of scalar registers to VGPR lanes
        // fell from 84 to 28 in the dense kernel).
        int zero;
        asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
        KernArgs* pk = (KernArgs*)((const __attribute__((address_space(4))) char*)&p + zero);
        attn_tile<kWide, kVT, false, kPartF32>(*pk, tile, chunk, chunks, slot, !planned, nullptr, false, -1, nullptr, nullptr, wave_first);
    }
}

// The work list of a packed varlen launch, built on the device from the
// segment offsets (the host does not have them) by one workgroup:
//   1. the query and key length of every segment (clamped as attn_tile
//      clamps them);
//   2. segments ordered by key length, longest first (ties: segment order;
//      up to kPlanSortMax segments, beyond that in segment order), so the
//      longest tiles run first and the last round holds the shortest;
//   3. the non-empty (segment, head, query tile) tiles in that order, the
//      heads and query tiles of one segment consecutive (they share K/V);
//   4. n_full = the whole rounds but the last (as for dense launches), and
//      the last round's tiles cut into key-range pieces (kQueuePieces, fewer
//      when a piece would hold under kQueueMinKeyTiles key tiles; one piece
//      writes the output itself), with merge slots for the split tiles;
//   5. the counts, and the tail counter zeroed.
constexpr int kPlanSortMax = 2048;

// Bound by latency (one workgroup, a chain of dependent steps), so every step
// is spread over 1,024 threads: prefix sums by wave shuffles, one thread per
// list entry, which finds its segment by bisection of the segments' first
// positions. 48 segments, 920 tiles: 22 us with 256 threads, sums through LDS
// and the segments' entries written one segment after another; 7.9 now.
constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over the workgroup's threads; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* buf, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(incl, off, 64);
        if (lane >= off) incl += up;
    }
    if (lane == 63) buf[wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        before += w < wave ? buf[w] : 0;
        all += buf[w];
    }
    *total = all;
    __syncthreads();
    return before + incl - v;
}

// Packed launches of short segments without a work list: one workgroup per CU
// runs tile after tile, and each tile issues the next one's Q loads and first
// K / V DMA during its own last two iterations, so the next tile starts with
// them in flight or landed instead of paying their latency (5-7 us against
// 1.5 us per key tile). Tiles [0, grid) start one per workgroup; every later
// one is claimed from the counter at p.persist_queue (tile grid + claim),
// two tiles ahead of its run, so the claim's latency passes during a tile and
// workgroups that drew short tiles take more of them.
// With p.persist_sort (segments of varied lengths, at most kPersistSegs) every
// workgroup first orders the segments by key length, longest first, and the
// tiles are claimed in that order without the ones past a segment's rows: the
// launch ends on the shortest tiles (in segment order the last claims could be
// the longest, and each missing tile cost a claim: 48 segments of 1 to 2,048
// rows at 5 heads 227 -> 214 us, 27 of 1 to 1,117 at 4 heads 78 -> 52). The order costs each workgroup about 2 us
// at its start, so equal lengths keep the segment order.
constexpr int kPersistSegs = 256;

__global__ __launch_bounds__(kThreads, 2) void attn_fwd_persist_kernel(AttnParams p) {
    __shared__ int claim;
    __shared__ int seg_key[kPersistSegs], seg_tiles[kPersistSegs];    // by segment
    __shared__ int seg_at[kPersistSegs], seg_base[kPersistSegs];      // by place in the order
    const int grid = (int)gridDim.x;
    const bool sorted = p.persist_sort != 0;
    int total = p.n_qtiles * p.heads * p.n_groups;
    if (sorted) {
        const int i = threadIdx.x, n = p.n_groups;  // n <= kPersistSegs (set by the launcher)
        if (i < n) {
            const int q0 = min(max(p.cu_q[i], 0), p.seqlen_q), k0 = min(max(p.cu_k[i], 0), p.seqlen_k);
            const int sq = min(max(p.cu_q[i + 1], q0), p.seqlen_q) - q0;
            seg_key[i] = min(max(p.cu_k[i + 1], k0), p.seqlen_k) - k0;
            seg_tiles[i] = min((sq + kBM - 1) / kBM, p.n_qtiles) * p.heads;
        }
        __syncthreads();
        if (i < n) {
            const int key = seg_key[i];
            int place = 0, base = 0;
            for (int j = 0; j < n; ++j) {
                const int kj = seg_key[j];
                const bool before = kj > key || (kj == key && j < i);
                place += before;
                base += before ? seg_tiles[j] : 0;
            }
            seg_at[place] = i;
            seg_base[place] = base;
        }
        __syncthreads();
        const int last = seg_at[n - 1];
        total = __builtin_amdgcn_readfirstlane(seg_base[n - 1] + seg_tiles[last]);
        if ((int)blockIdx.x >= total) return;
    }
    // Tile number of list position v: the last place whose tiles start at or
    // before it (segments without tiles share their successor's base).
    auto tile_of = [&](int v) __attribute__((always_inline)) {
        if (!sorted || v < 0) return v;
        const int lane = threadIdx.x & 63;
        int below = 0;
        for (int r = 0; r < p.n_groups; r += 64)
            below += __builtin_popcountll(__builtin_amdgcn_ballot_w64(r + lane < p.n_groups && seg_base[r + lane] <= v));
        const int place = below - 1;
        const int s = __builtin_amdgcn_readfirstlane(seg_at[place]);
        const int u = v - __builtin_amdgcn_readfirstlane(seg_base[place]);
        const int tq = __builtin_amdgcn_readfirstlane(seg_tiles[s]) / p.heads;
        return (s * p.heads + u / tq) * p.n_qtiles + u % tq;
    };
    // Segment bounds of tile t, loaded one tile ahead: they have landed when
    // the tile starts, and the next tile's by the time its loads are issued.
    // Read through the constant address space (nothing writes them during
    // the launch): scalar loads, which vector-memory waits do not count.
    using ConstInt = const __attribute__((address_space(4))) int;
    ConstInt* const cq = (ConstInt*)(uintptr_t)p.cu_q;
    ConstInt* const ck = (ConstInt*)(uintptr_t)p.cu_k;
    auto bounds = [&](int t, int* c) {
        const int s = t / p.n_qtiles / p.heads;
        c[0] = cq[s];
        c[1] = cq[s + 1];
        c[2] = ck[s];
        c[3] = ck[s + 1];
    };
    // Every wave reads the claim before thread 0 writes the next one.
    auto broadcast = [&](int c) {
        if (threadIdx.x == 0) claim = c;
        __syncthreads();
        const int v = __builtin_amdgcn_readfirstlane(claim);
        __syncthreads();
        return tile_of(grid + v < total ? grid + v : -1);
    };
    int t = tile_of(blockIdx.x);  // grid <= the tiles there can be
    int nt = broadcast(threadIdx.x == 0 ? atomicAdd(p.persist_queue, 1) : 0);
    bf16x8 qf[8];
    int cur[4], nxt[4];
    bool pre = false;
    bounds(t, cur);
    for (;;) {
        bounds(nt >= 0 ? nt : t, nxt);
        int c_after = 0;
        if (nt >= 0 && threadIdx.x == 0) c_after = atomicAdd(p.persist_queue, 1);
        // The arguments through an opaque address, as in the tail loop above.
        int zero;
        asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
        KernArgs* pk = (KernArgs*)((const __attribute__((address_space(4))) char*)&p + zero);
        pre = attn_tile<false, false, true>(*pk, t, -1, 1, -1, false, qf, pre, nt, cur, nxt);
        if (nt < 0) break;
        t = nt;
        nt = broadcast(c_after);
#pragma unroll
        for (int i = 0; i < 4; ++i) cur[i] = nxt[i];
    }
}

// Seg: where the per-segment arrays lie (4 * n_groups words).
template <typename Seg>
__device__ __forceinline__ void varlen_plan(const AttnParams& p, Seg segq, bool sorted, int* scan) {
    const int t = threadIdx.x;
    const int nseg = p.n_groups, heads = p.heads, nq = p.n_qtiles, cus = p.plan_cus;
    int* const info = p.vplan_w;
    int* const list = p.vlist_w;
    int* const pieces = p.vpieces_w;
    int* const merge = p.vmerge_w;
    const Seg segk = segq + nseg, order = segk + nseg, base = order + nseg;
    for (int i = t; i < nseg; i += kPlanThreads) {
        const int q0 = min(max(p.cu_q[i], 0), p.seqlen_q);
        const int k0 = min(max(p.cu_k[i], 0), p.seqlen_k);
        segq[i] = min(max(p.cu_q[i + 1], q0), p.seqlen_q) - q0;
        segk[i] = min(max(p.cu_k[i + 1], k0), p.seqlen_k) - k0;
    }
    __syncthreads();
    for (int i = t; i < nseg; i += kPlanThreads) {
        int r = i;
        if (sorted) {
            const int li = segk[i];
            r = 0;
            for (int j = 0; j < nseg; ++j) r += (segk[j] > li) | ((segk[j] == li) & (j < i));
        }
        order[r] = i;
    }
    __syncthreads();
    // Tiles of the segments in that order (query rows past n_qtiles tiles
    // are not computed: max_seqlen_q bounds every segment).
    int carry = 0;
    for (int c0 = 0; c0 < nseg; c0 += kPlanThreads) {
        const int r = c0 + t;
        const int cnt = r < nseg ? min((segq[order[r]] + kBM - 1) / kBM, nq) * heads : 0;
        int tot;
        const int off = block_scan(cnt, scan, &tot);
        if (r < nseg) base[r] = carry + off;
        carry += tot;
    }
    // Offsets that ascend give at most ub_tiles tiles; others are cut there.
    const int n_tiles = min(carry, p.ub_tiles);
    __syncthreads();
    // Place (in the order) of list position pos: the last r with base[r] <= pos
    // (empty segments share their successor's base).
    auto place = [&](int pos) {
        int lo = 0, hi = nseg - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (base[mid] <= pos) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    for (int i = t; i < n_tiles; i += kPlanThreads) {
        const int r = place(i), seg = order[r], u = i - base[r];
        const int tq = min((segq[seg] + kBM - 1) / kBM, nq);
        list[i] = (seg * heads + u / tq) * nq + u % tq;
    }
    const int n_full = n_tiles > cus ? (n_tiles - 1) / cus * cus : 0;
    const int n_last = n_tiles - n_full;
    int piece_carry = 0, merge_carry = 0;
    for (int c0 = 0; c0 < n_last; c0 += kPlanThreads) {
        const int i = c0 + t;
        int n = 0;
        if (i < n_last) {
            const int nkt = (segk[order[place(n_full + i)]] + kBN - 1) / kBN;
            n = kQueuePieces;
            while (n > 1 && nkt / n < kQueueMinKeyTiles) --n;
        }
        int ptot, mtot;
        const int poff = block_scan(n, scan, &ptot);
        const int moff = block_scan(n > 1 ? 1 : 0, scan, &mtot);
        if (i < n_last) {
            const int pos = n_full + i;
            const int ms = n > 1 ? merge_carry + moff : -1;
            for (int c = 0; c < n; ++c) {
                pieces[2 * (piece_carry + poff + c)] = pos;
                pieces[2 * (piece_carry + poff + c) + 1] = c | (n << 2) | ((ms + 1) << 5);
            }
            if (ms >= 0) {
                merge[2 * ms] = pos;
                merge[2 * ms + 1] = n;
            }
        }
        piece_carry += ptot;
        merge_carry += mtot;
    }
    if (t == 0) {
        info[kPlanTiles] = n_tiles;
        info[kPlanFull] = n_full;
        info[kPlanPieces] = piece_carry;
        info[kPlanMerges] = merge_carry;
        info[kPlanQueue] = 0;
    }
}

__global__ __launch_bounds__(kPlanThreads) void attn_varlen_plan_kernel(AttnParams p) {
    __shared__ int scan[kPlanThreads / 64];
    // Per-segment arrays: in LDS up to kPlanSortMax segments (the planner is
    // a chain of dependent accesses, so their latency is its time), in the
    // workspace beyond.
    __shared__ int lds_seg[4 * kPlanSortMax];
    if (p.n_groups <= kPlanSortMax)
        varlen_plan(p, (__attribute__((address_space(3))) int*)lds_seg, true, scan);
    else
        varlen_plan(p, p.vscratch, false, scan);
}

// d-major copy of V for the kVT form: vt holds, per (batch, head), 128 rows
// (head dims) of vt_rs bytes with keys contiguous, zero from seqlen_k to the
// next multiple of kBN. One workgroup moves a 64-key x 128-dim block through
// LDS: 16-byte row loads in, 16-byte dim-row stores out (8 lanes per 128-byte
// row). Rows are 65 dwords in LDS, so both phases are bank-conflict free.
__global__ __launch_bounds__(256) void attn_vt_kernel(AttnParams p) {
    __shared__ uint32_t blk[kBN * 65];
    const int t = threadIdx.x;
    const int h = blockIdx.y, b = blockIdx.z;
    // The dynamic tail's counter, for the attention kernel that follows on
    // the stream (instead of a launch of attn_queue_reset).
    if (p.queue != nullptr && t == 0 && blockIdx.x == 0 && h == 0 && b == 0) *p.queue = 0;
    // Block x moves keys [64x, 64x + 64) of the d-major layout. Dense: key k
    // of the sequence sits at k. Packed varlen: segment s starts at
    // vt_segment_start (its own rows, padded to a multiple of 64).
    const int k0 = blockIdx.x * kBN;
    int src0 = k0, src_end = p.seqlen_k;
    if (p.cu_k != nullptr) {
        // The grid covers every key of the rows; keys outside every segment
        // (padding, gaps) are written as zeros, so the attention kernel never
        // reads uninitialised memory past a segment's end.
        const int nseg = p.n_groups;
        int lo = 0, hi = nseg - 1;  // the last segment starting at or before k0
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (vt_segment_start(min(max(p.cu_k[mid], 0), p.seqlen_k), mid) <= k0) lo = mid; else hi = mid - 1;
        }
        const int s0 = min(max(p.cu_k[lo], 0), p.seqlen_k);
        const int s1 = min(max(p.cu_k[lo + 1], s0), p.seqlen_k);
        const int v0 = vt_segment_start(s0, lo);
        src0 = s0 + (k0 - v0);
        src_end = k0 >= v0 ? s1 : src0;  // before the first segment's start: zeros
    }
    const char* src = (const char*)p.v + 2 * (b * p.v_sb + h * p.v_sh);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = i * 16 + (t >> 4), c = t & 15;
        i32x4 x = i32x4{0, 0, 0, 0};
        if (src0 + key < src_end) x = *(const i32x4*)(src + (int64_t)(src0 + key) * p.v_rs + c * 16);
        uint32_t* row = blk + key * 65 + c * 4;
        row[0] = (uint32_t)x.x;
        row[1] = (uint32_t)x.y;
        row[2] = (uint32_t)x.z;
        row[3] = (uint32_t)x.w;
    }
    __syncthreads();
    char* dst = (char*)p.vt + 2 * (b * p.vt_sb + h * p.vt_sh + (int64_t)k0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = i * 32 + (t >> 3), kc = t & 7;
        const int sh = (d & 1) * 16;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = blk[(8 * kc + 2 * j) * 65 + (d >> 1)] >> sh;
            const uint32_t up = blk[(8 * kc + 2 * j + 1) * 65 + (d >> 1)] >> sh;
            w[j] = (lo & 0xffffu) | (up << 16);
        }
        *(i32x4*)(dst + (int64_t)d * p.vt_rs + kc * 16) = i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    }
}

// Zeroes the dynamic tail's counter (a kernel, not a memset, so that the
// launch can be captured in a graph).
__global__ void attn_queue_reset(int* queue) {
    if (threadIdx.x == 0) *queue = 0;
}

}  // namespace

int attn_fwd_unit_rows() { return kUnitRows; }
int attn_fwd_block_m() { return kBM; }
int attn_fwd_persist_max_segments() { return kPersistSegs; }
int attn_fwd_persist_max_rows() { return kPersistMaxQTiles * kBM; }
int attn_fwd_tail_pieces() { return kQueuePieces; }
int64_t attn_fwd_piece_bytes(bool f32) { return (int64_t)kBM * (kD * (f32 ? 4 : 2) + 4); }
int attn_fwd_block_n() { return kBN; }
int attn_fwd_window_rows() { return kWindowRows > kBM ? kWindowRows : kBM; }
int attn_fwd_row_margin() { return kBM + kBN * (2 * kStages + 2); }

// Expected time of the jobs (tiles or pieces of kt key tiles) of the last rounds
// of a launch: their fixed part and their key tiles, slower the more CUs are
// busy (power).
static double round_us(int64_t jobs, double kt, int cus) {
    const double busy = jobs < cus ? (double)jobs / (double)cus : 1.0;
    return (double)((jobs + cus - 1) / cus) * (kTileUs + kt * (1.0 + 0.6 * busy));
}

// Expected time of whole tiles, the last round cut where that is shorter.
static double tiles_us(int64_t tiles, int64_t key_tiles, int cus) {
    const int64_t full = (tiles - 1) / cus * cus, rest = tiles - full;
    const int n = plan_attn_last_round(tiles, key_tiles, cus, INT64_MAX).split_n;
    return (double)(full / cus) * round_us(cus, (double)key_tiles, cus) +
           (n > 0 ? round_us(rest * n, (double)key_tiles / n, cus) + kPiecesUs : round_us(rest, (double)key_tiles, cus));
}

bool attn_rag_pays(int64_t whole, int64_t units, int64_t keys, int cus) {
    if (cus <= 0) return false;
    if (whole + units <= cus) return true;  // all at once, as the tiles would be
    // The units read every head's K and V again, which the ragged tiles have
    // from the L2 beside their neighbours (512 bytes a key at about 3.4 TB/s
    // while the tiles run).
    const int64_t kt = (keys + kBN - 1) / kBN;
    return tiles_us(whole + units, kt, cus) - tiles_us(whole, kt, cus) > 1.5e-4 * (double)units * (double)keys;
}

int attn_rag_blocks(int64_t tiles, int64_t units, int64_t keys, int cus) {
    // The units run one after another on the CUs that the last round of tiles
    // leaves idle where they have the time for it, else one per workgroup. (As
    // one workgroup each they would wait for a CU of the shader engine whose
    // turn it is, though others are idle: 40 units beside 240 tiles took 13 us
    // longer than 36 beside 216.)
    const int64_t idle = cus > 0 ? (cus - tiles % cus) % cus : 0;
    const double tile_us = kTileUs + 1.6 * (double)((keys + kBN - 1) / kBN);
    const double unit_us = 5.0 + 1.6 * (double)((keys + kUnitKeys * kWaves - 1) / (kUnitKeys * kWaves));
    return (int)(idle * (int64_t)(tile_us / unit_us) >= units && idle < units ? idle : units);
}

SplitPlan plan_attn_split(int64_t tiles, int64_t key_tiles, int cus, int64_t max_workspace) {
    SplitPlan plan{(int32_t)tiles, 0, 0, 0, 0, 0, 0};
    if (cus < 8 || cus % 8 != 0 || tiles <= 0) return plan;
    const int64_t piece_bytes = attn_fwd_piece_bytes(false);  // bf16 partial O and fp32 LSE of a piece's rows
    if (tiles > cus) {
        // Dynamic tail: the whole rounds but the last run as they are; the
        // last round's tiles become kQueuePieces key-range pieces each, taken
        // from a counter by cus workgroups (at most) as CUs free up. Pieces
        // keep at least kQueueMinKeyTiles key tiles, so the pipeline's fill
        // and drain stay small against a piece; fewer pieces are cut when
        // their partial results would not fit in max_workspace.
        const int64_t full = (tiles - 1) / cus * cus, rest = tiles - full;
        auto bytes = [&](int n) { return ((int64_t)n * rest * piece_bytes + 255) / 256 * 256 + 256; };
        int n = kQueuePieces;
        while (n > 1 && (key_tiles / n < kQueueMinKeyTiles || bytes(n) > max_workspace)) --n;
        if (n < 2) return plan;
        plan.n_full = (int32_t)full;
        plan.split_n = n;
        plan.split_tiles = (int32_t)rest;
        plan.queue_blocks = (int32_t)(rest * n < cus ? rest * n : cus);
        plan.queue_offset = ((int64_t)n * rest * piece_bytes + 255) / 256 * 256;
        plan.workspace_bytes = bytes(n);
        return plan;
    }
    // One partial round: its tiles are cut into n key-range pieces when that
    // shortens the round (n <= 8, at least one key tile per piece):
    // ceil(tiles * n / cus) / n. The chip is power-bound under this kernel:
    // a round that keeps 70% or more of the CUs busy runs at a higher clock
    // and loses little, and splitting it does not pay for the pieces and the
    // merge.
    if (tiles * 10 >= (int64_t)cus * 7) return plan;
    double best = 1.0;
    int best_n = 0;
    for (int n = 2; n <= 8 && n <= key_tiles; ++n) {
        if ((int64_t)n * tiles * piece_bytes > max_workspace) break;
        const double cost = (double)((tiles * n + cus - 1) / cus) / n;
        if (cost < best - 0.05) {
            best = cost;
            best_n = n;
        }
    }
    if (best_n == 0) return plan;
    plan.n_full = 0;
    plan.split_n = best_n;
    plan.split_tiles = (int32_t)tiles;
    plan.workspace_bytes = (int64_t)best_n * tiles * piece_bytes;
    return plan;
}

SplitPlan plan_attn_last_round(int64_t tiles, int64_t key_tiles, int cus, int64_t max_workspace) {
    SplitPlan plan{(int32_t)tiles, 0, 0, 0, 0, 0, 0};
    if (cus < 8 || cus % 8 != 0 || tiles <= cus) return plan;
    const int64_t piece_bytes = attn_fwd_piece_bytes(true);
    const int64_t full = (tiles - 1) / cus * cus, rest = tiles - full;
    auto bytes = [&](int n) { return ((int64_t)n * rest * piece_bytes + 255) / 256 * 256 + 256; };
    // Pieces pay where they fill a last round that would leave CUs idle, by the
    // expected time, with what they cost besides (the counter's reset, the
    // merge; 3-4 us of it for partial results in fp32 against bf16). Measured
    // (us, whole -> pieces): 24 heads of 4,096 x 4,096 218 -> 210, 40 of 2,048 x
    // 2,048 105 -> 101, 20 of 3,500 x 3,500 166 -> 136, 9 of 7,424 x 6,000 271
    // -> 195; 8 of 10,240 x 1,024 58 -> 60 (bf16), which the rule leaves whole.
    int n = 0;
    double best = round_us(rest, (double)key_tiles, cus) - 2.0;
    for (int c = 2; c <= kMaxPieces && key_tiles / c >= 2 && bytes(c) <= max_workspace; ++c) {
        const double us = round_us(rest * c, (double)key_tiles / c, cus) + kPiecesUs;
        if (us < best) {
            best = us;
            n = c;
        }
    }
    if (n == 0) return plan;
    plan.n_full = (int32_t)full;
    plan.split_n = n;
    plan.split_tiles = (int32_t)rest;
    plan.queue_blocks = (int32_t)(rest * n < cus ? rest * n : cus);
    plan.queue_offset = ((int64_t)n * rest * piece_bytes + 255) / 256 * 256;
    plan.workspace_bytes = bytes(n);
    plan.part_f32 = 1;
    return plan;
}

hipError_t attn_static_scratch(void** ptr) {
    // Looked up once per device (with that device current), then cached.
    static std::atomic<void*> cache[64];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev >= 0 && dev < 64) {
        void* hit = cache[dev].load(std::memory_order_acquire);
        if (hit != nullptr) {
            *ptr = hit;
            return hipSuccess;
        }
    }
    void* addr = nullptr;
    e = hipGetSymbolAddress(&addr, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return e;
    if (dev >= 0 && dev < 64) cache[dev].store(addr, std::memory_order_release);
    *ptr = addr;
    return hipSuccess;
}

hipError_t launch_attn_fwd(const AttnParams& p, hipStream_t stream) {
    if (p.n_units > 0) {
        // Packed: no more than the rows and a part of a unit per segment give.
        int64_t units = (int64_t)p.n_units * p.heads * p.n_groups;
        const int64_t rows = p.heads * ((int64_t)p.seqlen_q / kUnitRows + p.n_groups);
        if (p.cu_q != nullptr && rows < units) units = rows;
        hipLaunchKernelGGL(attn_short_kernel, dim3((unsigned)units), dim3(kThreads), 0, stream, p);
        return hipGetLastError();
    }
    const int64_t tiles = (int64_t)p.n_qtiles * p.heads * p.n_groups;
    if (tiles <= 0) return hipSuccess;
    int64_t blocks = tiles;
    if (p.vplan != nullptr) {
        // The list, its pieces and the d-major V offsets first.
        hipLaunchKernelGGL(attn_varlen_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
        blocks = (int64_t)p.ub_tiles + p.plan_cus;
    } else if (p.queue != nullptr) {
        // With a d-major V copy the transpose kernel zeroes the counter.
        if (p.vt == nullptr) hipLaunchKernelGGL(attn_queue_reset, dim3(1), dim3(64), 0, stream, p.queue);
        blocks = (int64_t)p.n_full + p.queue_blocks;
    } else if (p.split_n != 0) {
        blocks = (int64_t)p.n_full + (int64_t)p.split_n * p.split_tiles;
    }
    if (p.vt != nullptr) {
        // Dense: the keys of the sequence; varlen: every key of the padded rows.
        const int64_t vt_tiles = (p.seqlen_k + kBN - 1) / kBN + (p.cu_k != nullptr ? p.n_groups : 0);
        const dim3 tgrid((unsigned)vt_tiles, (unsigned)p.heads, (unsigned)(p.cu_k != nullptr ? 1 : p.n_groups));
        hipLaunchKernelGGL(attn_vt_kernel, tgrid, dim3(256), 0, stream, p);
    }
    const dim3 block(kThreads);
    // Persistent only for short segments (at most kPersistMaxQTiles query
    // tiles each), where a tile's fixed cost is a large share of it.
    if (p.cu_q != nullptr && p.vplan == nullptr && !p.wide && p.vt == nullptr && p.split_n == 0 &&
        p.queue == nullptr && p.persist_queue != nullptr && p.persist_blocks > 0 && p.n_qtiles <= kPersistMaxQTiles) {
        const int64_t n = blocks < p.persist_blocks ? blocks : p.persist_blocks;
        hipLaunchKernelGGL(attn_queue_reset, dim3(1), dim3(64), 0, stream, p.persist_queue);
        hipLaunchKernelGGL(attn_fwd_persist_kernel, dim3((unsigned)n), block, 0, stream, p);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)(blocks + p.rag_blocks));
    if (p.wide && p.vt != nullptr)
        hipLaunchKernelGGL((attn_fwd_kernel<true, true>), grid, block, 0, stream, p);
    else if (p.wide)
        hipLaunchKernelGGL((attn_fwd_kernel<true, false>), grid, block, 0, stream, p);
    else if (p.vt != nullptr)
        hipLaunchKernelGGL((attn_fwd_kernel<false, true>), grid, block, 0, stream, p);
    else if (p.part_f32 != 0)
        hipLaunchKernelGGL((attn_fwd_kernel<false, false, true>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((attn_fwd_kernel<false, false>), grid, block, 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.vplan != nullptr) {
        // Every possible merge slot (at most plan_cus split tiles); slots past
        // the plan's count exit.
        const dim3 merge_grid((unsigned)(p.plan_cus * (kBM / kMergeRows)));
        hipLaunchKernelGGL(attn_merge_kernel<4>, merge_grid, dim3(256), 0, stream, p);
        return hipGetLastError();
    }
    if (p.split_n == 0) return e;
    const dim3 merge_grid((unsigned)(p.split_tiles * (kBM / kMergeRows)));
    if (p.part_f32 != 0)
        hipLaunchKernelGGL((attn_merge_kernel<8, true>), merge_grid, dim3(256), 0, stream, p);
    else if (p.split_n <= 4)
        hipLaunchKernelGGL(attn_merge_kernel<4>, merge_grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(attn_merge_kernel<8>, merge_grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace h3a
