// One step's metadata built on the GPU from the requests' lengths: block tables, slot mapping,
// positions and the split-KV work list of the static step layout.
//
// The host-built step (gkv_upload_step) packs every request's whole table, validates and plans on
// the CPU and copies the result, for tables that change by one entry every block_size tokens.
// Here the caller's tables stay on the device and one launch writes what the step adds.  Request
// b with c tokens stored and n to add, block size s:
//   first page to open o = ceil(c / s), pages after the step a = ceil((c + n) / s),
//   table[o + j] = new_blocks[F + j] for j < a - o, F = sum of (a - o) over the requests before b,
//   its tokens are rows C .. C + n of the step, C = sum of n over the requests before b,
//   token C + i: position p = c + i, slot = table[p / s] * s + p % s.
// A request is left out (error bit, its rows' slots -1, its context 0 so that the decode leaves its
// output alone, its tables as they were) when its lengths are negative, reach past its table row,
// need blocks past the end of new_blocks or rows past max_tokens.
//
// The work list is the host planner's, entry for entry (plan_work_into, step.cpp).  The host walks
// the flattened stream of all (request, kv head) segments; here every worker and every segment
// finds its own cuts: worker w covers [floor(w T / n), floor((w + 1) T / n)) of the T units, so the
// worker that holds unit u is ceil((u + 1) n / T) - 1, and slots and pieces are numbered by scans.
//
// Latency-bound: the bytes are a few per request and 12 per token.  So there is one launch and no
// wait between its blocks: each block repeats the scan over the requests (at most 4096, from L2), the
// first few plan, the others write tables, slots and positions.
//
// Measured, replayed in a graph: 64 decodes of 4 kv heads 6.5 us, 1024 decodes 9.0 us, 40 prompts of
// together 48,000 tokens 6.5 us.  It is the chain of scan, cuts and numbering: with 64-bit products, binary
// searches and five barriers a scan it took 16 to 24 us.
#include "gkv_device.cuh"
#include "kernels.h"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kSegInSmem = 12288;  // segments whose prefixes a planning block keeps in shared memory

// Rows and pages only ever matter up to 2^31 - 1: sums stop there.
__device__ __forceinline__ uint32_t add_to_limit(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

// What the scan over the requests adds up.
struct Counts {
    uint32_t rows, pages;  // at most 2^31 - 1 each
    uint32_t live;         // requests with units
    int64_t units;
    static __device__ __forceinline__ Counts plus(const Counts& a, const Counts& b) {
        return Counts{add_to_limit(a.rows, b.rows), add_to_limit(a.pages, b.pages), a.live + b.live, a.units + b.units};
    }
    static __device__ __forceinline__ Counts up(const Counts& a, int o) {
        return Counts{__shfl_up_sync(~0u, a.rows, o), __shfl_up_sync(~0u, a.pages, o), __shfl_up_sync(~0u, a.live, o),
                      __shfl_up_sync(~0u, a.units, o)};
    }
    static __device__ __forceinline__ Counts at(const Counts& a, int l) {
        return Counts{__shfl_sync(~0u, a.rows, l), __shfl_sync(~0u, a.pages, l), __shfl_sync(~0u, a.live, l),
                      __shfl_sync(~0u, a.units, l)};
    }
};
// Pieces of segments, and three counts of the split ones in one word: merge entries, long ones,
// partial slots (below 2^20, 2^20, 2^24: at most 2^20 segments, and a slot per worker and segment).
struct Splits {
    uint32_t pieces;
    uint64_t split;
    static __device__ __forceinline__ Splits plus(const Splits& a, const Splits& b) { return Splits{a.pieces + b.pieces, a.split + b.split}; }
    static __device__ __forceinline__ Splits up(const Splits& a, int o) {
        return Splits{__shfl_up_sync(~0u, a.pieces, o), __shfl_up_sync(~0u, a.split, o)};
    }
    static __device__ __forceinline__ Splits at(const Splits& a, int l) {
        return Splits{__shfl_sync(~0u, a.pieces, l), __shfl_sync(~0u, a.split, l)};
    }
    static __device__ __forceinline__ Splits of(int pieces) {
        if (pieces <= 1) return Splits{static_cast<uint32_t>(pieces), 0};
        return Splits{static_cast<uint32_t>(pieces),
                      1ull | (pieces > kWarpMergeMaxSlots ? 1ull << 20 : 0ull) | (static_cast<uint64_t>(pieces) << 40)};
    }
    __device__ __forceinline__ int merges() const { return static_cast<int>(split & 0xfffff); }
    __device__ __forceinline__ int longs() const { return static_cast<int>((split >> 20) & 0xfffff); }
    __device__ __forceinline__ int slots() const { return static_cast<int>(split >> 40); }
};

// Exclusive prefix of x over the block, `carry` included; carry grows by the sum.  Calls in a row use
// the two halves of `part` [2][kWarps] in turn, so one barrier each is enough: a half is written again
// only behind the barrier of the call in between.
template <typename T>
__device__ __forceinline__ T block_scan(const T& x, T& carry, T* part, int& turn) {
    static_assert(kWarps == 32, "one partial sum per lane");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = T::up(inc, o);
        if (lane >= o) inc = T::plus(y, inc);
    }
    T before = T::up(inc, 1);
    if (lane == 0) before = T{};
    T* p = part + turn * kWarps;
    turn ^= 1;
    if (lane == 31) p[warp] = inc;
    __syncthreads();
    T s = p[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = T::up(s, o);
        if (lane >= o) s = T::plus(y, s);
    }
    const T base = T::at(s, warp > 0 ? warp - 1 : 0);
    const T mine = warp > 0 ? T::plus(carry, base) : carry;
    carry = T::plus(carry, T::at(s, 31));
    return T::plus(mine, before);
}

__device__ __forceinline__ int64_t chunks_in(int64_t ctx, int bs) {
    const int cpp = (bs + kDecodeChunk - 1) / kDecodeChunk;
    const int c = static_cast<int>(ctx), full = c / bs;
    return static_cast<int64_t>(full) * cpp + (c - full * bs + kDecodeChunk - 1) / kDecodeChunk;
}

struct Request {
    uint32_t ctx, n;   // as given, negative ones as 0
    uint32_t old_pages, opened;
    bool fits;         // lengths valid and within the table row
};

__device__ __forceinline__ Request load_request(const StepBuildArgs& a, int b) {
    Request r;
    const int c = __ldg(a.ctx_lens + b), n = __ldg(a.new_lens + b);
    r.ctx = c > 0 ? c : 0;
    r.n = n > 0 ? n : 0;
    const uint32_t end = r.ctx + r.n;  // below 2^32
    r.fits = c >= 0 && n >= 0 && end <= 0x7fffffffu && end <= a.table_stride * a.block_size;
    const uint32_t bs = a.block_size;
    r.old_pages = r.ctx / bs + (r.ctx % bs != 0);
    r.opened = r.fits ? end / bs + (end % bs != 0) - r.old_pages : 0;
    return r;
}

// Last index b in [0, n) with pre[b] <= x; pre is non-decreasing and pre[0] <= x.
template <typename T>
__device__ __forceinline__ int last_at_most(const T* pre, int n, T x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Whether a request whose rows start at row0 and whose new pages start at page0 is in the step.
__device__ __forceinline__ bool served(const StepBuildArgs& a, const Request& r, uint32_t row0, uint32_t page0) {
    return r.fits && (r.n == 0 || row0 + r.n <= static_cast<uint32_t>(a.max_tokens)) &&
           (r.opened == 0 || page0 + r.opened <= static_cast<uint32_t>(a.n_new_blocks));
}

// ---- the work list ------------------------------------------------------------------------

// The stream of units over the live requests (those with a context): request k's head h spans units
// [pre[k] + h * span, ... + span), span = kSegmentCost + its chunks, pre[k + 1] = pre[k] + H span.
// Quotients come from estimates in 32-bit floating point, put right by one exact product to each
// side: they are below 2^14 (workers) and 2^10 (heads), so an estimate is off by less than one.
struct Units {
    const uint32_t* pre;  // [live + 1]
    int live, H, n;       // n: workers
    uint32_t total, q, r; // total = q * n + r, below 2^31
    float n_over_total, inv_n, inv_H;

    // first unit of worker w: floor(w * total / n)
    __device__ __forceinline__ uint32_t begin(int w) const {
        const uint32_t x = r * static_cast<uint32_t>(w);  // below 2^28
        uint32_t e = static_cast<uint32_t>(static_cast<float>(x) * inv_n);
        e -= e * n > x;
        e += (e + 1) * n <= x;
        return q * static_cast<uint32_t>(w) + e;
    }
    // the worker that holds unit u: the last w with floor(w * total / n) <= u, i.e. w * total < (u + 1) n
    __device__ __forceinline__ int worker_of(uint32_t u) const {
        uint32_t w = static_cast<uint32_t>(static_cast<float>(u) * n_over_total);
        const uint64_t end = (static_cast<uint64_t>(u) + 1) * n, t = total;
        w -= w * t >= end;
        w += (w + 1) * t < end;
        return static_cast<int>(w);
    }
    __device__ __forceinline__ uint32_t span(int k) const {
        const uint32_t s = pre[k + 1] - pre[k];
        uint32_t e = static_cast<uint32_t>(static_cast<float>(s) * inv_H);  // a multiple of H: find the exact quotient
        while (e * H > s) --e;
        while (e * H < s) ++e;
        return e;
    }
    // segment of unit u: live request and head, and the segment's first unit
    __device__ __forceinline__ void segment_of(uint32_t u, int& k, int& h, uint32_t& s0, uint32_t& sp) const {
        int lo = 0, hi = live;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= u) lo = mid;
            else hi = mid;
        }
        k = lo;
        sp = span(lo);
        const uint32_t in = u - pre[lo];
        uint32_t e = static_cast<uint32_t>(__fdividef(static_cast<float>(in), static_cast<float>(sp)));
        e -= e * static_cast<uint64_t>(sp) > in;
        e += (e + 1) * static_cast<uint64_t>(sp) <= in;
        h = static_cast<int>(e);
        s0 = pre[lo] + e * sp;
    }
    // pieces of a segment that starts at unit s0: workers with units in [s0 + cost, s0 + span); one unit
    // each when there are fewer units than workers
    __device__ __forceinline__ int pieces(uint32_t s0, uint32_t sp) const {
        return total >= static_cast<uint32_t>(n) ? worker_of(s0 + sp - 1) - worker_of(s0 + kSegmentCost) + 1 : static_cast<int>(sp - kSegmentCost);
    }
    // pieces of it that belong to workers before w, whose first unit lo lies in the segment
    __device__ __forceinline__ int pieces_before(uint32_t s0, int w, uint32_t lo) const {
        if (lo <= s0 + static_cast<uint32_t>(kSegmentCost)) return 0;
        return total >= static_cast<uint32_t>(n) ? w - worker_of(s0 + kSegmentCost) : static_cast<int>(lo - s0 - kSegmentCost);
    }
};

// Planning block `part_no`: 0 writes the merge entries and the header, part_no >= 1 the pieces of
// workers (part_no - 1) * kThreads ...  Each goes over all segments first, for the prefixes.
__device__ void plan(const StepBuildArgs& a, const Units& u, const int32_t* id, int32_t* smem_seg, Splits* part, int part_no,
                     int n_tokens) {
    auto at = [&](int off) { return reinterpret_cast<int32_t*>(a.meta + off); };
    static_assert(kFusedMergeMaxSlots == 0, "the list below defers every merge");
    const int H = u.H, n_seg = u.live * H;
    // by segment: first partial slot (-1 for a segment in one piece), pieces before it.  Beyond the shared
    // memory, in the pool's scratch: every block writes the same values there and reads its own.
    int32_t* seg_slot = n_seg <= kSegInSmem ? smem_seg : a.scratch;
    int32_t* seg_piece = n_seg <= kSegInSmem ? smem_seg + n_seg : a.scratch + n_seg;
    int32_t* long_before = a.scratch + 2 * static_cast<int64_t>(a.batch) * H;  // by merge entry
    int turn = 0;
    Splits sum{};
    for (int base = 0; base < n_seg; base += kThreads) {
        const int s = base + static_cast<int>(threadIdx.x);
        int pieces = 0, k = 0, h = 0;
        if (s < n_seg) {
            k = s / H;
            h = s - k * H;
            const uint32_t sp = u.span(k);
            pieces = u.pieces(u.pre[k] + h * sp, sp);
        }
        const Splits x = block_scan(Splits::of(pieces), sum, part, turn);
        if (s < n_seg) {
            seg_slot[s] = pieces > 1 ? x.slots() : -1;
            seg_piece[s] = static_cast<int32_t>(x.pieces);
            if (part_no == 0 && pieces > 1) {
                const int m = x.merges();
                at(a.off_mseg)[m] = id[k] * H + h;
                at(a.off_ms0)[m] = x.slots();
                at(a.off_mns)[m] = pieces;
                long_before[m] = x.longs();
            }
        }
    }
    __syncthreads();
    if (part_no == 0) {
        // the deferred list: every split segment, the long ones first, each kind in order
        for (int m = static_cast<int>(threadIdx.x); m < sum.merges(); m += kThreads) {
            const int lb = long_before[m];
            at(a.off_mdef)[at(a.off_mns)[m] > kWarpMergeMaxSlots ? lb : sum.longs() + m - lb] = m;
        }
        if (threadIdx.x == 0) {
            at(a.off_wbeg)[a.n_workers] = static_cast<int32_t>(sum.pieces);
            int32_t* hd = at(0);
            hd[kHdrTok] = n_tokens;
            hd[kHdrBatch] = a.batch;
            hd[kHdrMaxBlocks] = static_cast<int32_t>(a.table_stride);
            hd[kHdrSlots] = sum.slots();
            hd[kHdrMerge] = sum.merges();
            hd[kHdrDeferred] = sum.merges();
            hd[kHdrDeferredLong] = sum.longs();
            hd[kHdrWorkers] = a.n_workers;
            hd[kHdrTables] = 0;
            hd[kHdrCtx] = a.off_ctx;
            hd[kHdrPseg] = a.off_pseg;
            hd[kHdrPc0] = a.off_pc0;
            hd[kHdrPc1] = a.off_pc1;
            hd[kHdrPslot] = a.off_pslot;
            hd[kHdrPmerge] = a.off_pmerge;
            hd[kHdrWbeg] = a.off_wbeg;
            hd[kHdrMseg] = a.off_mseg;
            hd[kHdrMs0] = a.off_ms0;
            hd[kHdrMns] = a.off_mns;
            hd[kHdrMdef] = a.off_mdef;
            *reinterpret_cast<uint64_t*>(hd + kHdrTablesPtr) = reinterpret_cast<uint64_t>(a.tables);
        }
        return;
    }
    const int w = (part_no - 1) * kThreads + static_cast<int>(threadIdx.x);
    if (w >= a.n_workers) return;
    if (u.total == 0) {
        at(a.off_wbeg)[w] = 0;
        return;
    }
    const uint32_t lo = u.begin(w), hi = u.begin(w + 1);
    if (lo >= u.total) {  // workers behind the last unit (fewer units than workers)
        at(a.off_wbeg)[w] = static_cast<int32_t>(sum.pieces);
        return;
    }
    int k, h;
    uint32_t s0, sp;
    u.segment_of(lo, k, h, s0, sp);
    const int before = u.pieces_before(s0, w, lo);
    int p = seg_piece[k * H + h] + before;
    at(a.off_wbeg)[w] = p;
    // from the worker's first segment to the one its range ends in; a range that ends inside a segment's
    // overhead has no piece of it, nor has a worker without a unit
    for (int nth = before; lo < hi && s0 < hi && hi > s0 + static_cast<uint32_t>(kSegmentCost); nth = 0, ++p) {
        const int first = seg_slot[k * H + h];
        at(a.off_pseg)[p] = id[k] * H + h;
        at(a.off_pc0)[p] = lo > s0 + static_cast<uint32_t>(kSegmentCost) ? static_cast<int32_t>(lo - s0 - kSegmentCost) : 0;
        at(a.off_pc1)[p] = static_cast<int32_t>(min(hi, s0 + sp) - s0 - kSegmentCost);
        at(a.off_pslot)[p] = first < 0 ? -1 : first + nth;
        at(a.off_pmerge)[p] = first < 0 ? -1 : -2;
        s0 += sp;
        if (++h == H) {
            h = 0;
            if (++k == u.live) break;
            sp = u.span(k);
        }
    }
}

// The scan over the requests: calls item(b, request, in the step, sums before it) for each, in rounds
// of a block's threads, and returns the sums.  Whether a request is in the step depends on the rows and
// pages before it, and its units on that: they are counted as if nothing passed a limit, and once more
// where something does.
template <typename F>
__device__ __forceinline__ Counts scan_requests(const StepBuildArgs& a, Counts* part, int& turn, F item) {
    Counts sum{};
    for (int base = 0; base < a.batch; base += kThreads) {
        const int b = base + static_cast<int>(threadIdx.x);
        Request r{};
        if (b < a.batch) r = load_request(a, b);
        const bool counted = b < a.batch && r.fits;
        int64_t chunks = counted ? chunks_in(r.ctx + r.n, a.block_size) : 0;
        const Counts was = sum;
        Counts at = block_scan(Counts{r.n, r.opened, chunks > 0, chunks > 0 ? chunks + kSegmentCost : 0}, sum, part, turn);
        bool ok = counted;
        if (sum.rows > static_cast<uint32_t>(a.max_tokens) || sum.pages > static_cast<uint32_t>(a.n_new_blocks)) {  // the same for all threads
            ok = counted && served(a, r, at.rows, at.pages);
            if (!ok) chunks = 0;
            Counts again = was;
            const Counts ua = block_scan(Counts{0, 0, chunks > 0, chunks > 0 ? chunks + kSegmentCost : 0}, again, part, turn);
            at.live = ua.live;
            at.units = ua.units;
            sum.live = again.live;
            sum.units = again.units;
        }
        if (b < a.batch) item(b, r, ok, at);
    }
    return sum;
}

__global__ void __launch_bounds__(kThreads, 1) step_build_kernel(const StepBuildArgs a, const int n_plan) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Counts part[2 * kWarps];
    __shared__ Splits splits[2 * kWarps];
    __shared__ int used_blocks, left_out;
    const int B = a.batch, H = a.heads_kv;
    int turn = 0;

    if (static_cast<int>(blockIdx.x) < n_plan) {
        // ---- a planning block: units and ids of the live requests, then its part of the work list ----
        uint32_t* pre = reinterpret_cast<uint32_t*>(smem);
        int32_t* id = reinterpret_cast<int32_t*>(pre + B + 1);
        int32_t* seg = id + B + 1;
        const Counts sum = scan_requests(a, part, turn, [&](int b, const Request& r, bool ok, const Counts& at) {
            const uint32_t ctx = ok ? r.ctx + r.n : 0;
            if (ctx > 0) {
                pre[at.live] = static_cast<uint32_t>(at.units * H);
                id[at.live] = b;
            }
            if (blockIdx.x == 0) reinterpret_cast<int32_t*>(a.meta + a.off_ctx)[b] = static_cast<int32_t>(ctx);
        });
        int live = static_cast<int>(sum.live);
        int64_t total = sum.units * H;
        __syncthreads();
        if (total >= int64_t{1} << 31) {  // more than the work list counts: nothing of the step is decoded
            for (int b = static_cast<int>(threadIdx.x); b < B && blockIdx.x == 0; b += kThreads)
                reinterpret_cast<int32_t*>(a.meta + a.off_ctx)[b] = 0;
            if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, kErrBadStep);
            total = 0;
            live = 0;
        }
        if (threadIdx.x == 0) pre[live] = static_cast<uint32_t>(total);
        __syncthreads();
        const uint32_t t = static_cast<uint32_t>(total), n = a.n_workers;
        const Units u{pre, live, H, a.n_workers, t, t / n, t % n, static_cast<float>(n) / static_cast<float>(t > 0 ? t : 1),
                      1.f / static_cast<float>(n), 1.f / static_cast<float>(H)};
        plan(a, u, id, seg, splits, blockIdx.x, min(static_cast<int>(sum.rows), a.max_tokens));
        return;
    }

    // ---- the other blocks: tables, rows and what there is one of per request ----
    uint32_t* row_pre = reinterpret_cast<uint32_t*>(smem);
    uint32_t* page_pre = row_pre + B + 1;
    const int nth = static_cast<int>(blockIdx.x) - n_plan;
    if (threadIdx.x == 0) used_blocks = left_out = 0;
    __syncthreads();
    const Counts sum = scan_requests(a, part, turn, [&](int b, const Request& r, bool ok, const Counts& at) {
        row_pre[b] = at.rows;
        page_pre[b] = at.pages;
        if (nth != 0) return;
        if (a.cu_new) a.cu_new[b] = static_cast<int32_t>(at.rows);
        if (a.ctx_out) a.ctx_out[b] = static_cast<int32_t>(ok ? r.ctx + r.n : r.ctx);
        if (ok && r.opened > 0) atomicMax(&used_blocks, static_cast<int>(at.pages + r.opened));
        if (!ok) left_out = 1;
    });
    __syncthreads();
    if (nth == 0 && threadIdx.x == 0) {
        if (a.cu_new) a.cu_new[B] = static_cast<int32_t>(sum.rows);
        if (a.counts) {
            a.counts[0] = static_cast<int32_t>(sum.rows);
            a.counts[1] = used_blocks;
        }
        if (left_out) atomicOr(a.err, kErrBadStep);
    }
    const uint32_t bs = a.block_size;
    const int stride = (static_cast<int>(gridDim.x) - n_plan) * kThreads;
    const int me = nth * kThreads + static_cast<int>(threadIdx.x);
    // opened pages into the tables
    const int n_pages = min(static_cast<int>(sum.pages), a.n_new_blocks);
    for (int j = me; j < n_pages; j += stride) {
        const int b = last_at_most<uint32_t>(page_pre, B, j);
        const Request r = load_request(a, b);
        if (!served(a, r, row_pre[b], page_pre[b])) continue;
        const int32_t id = __ldg(a.new_blocks + j);
        if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.total_blocks)) atomicOr(a.err, kErrBadBlock);
        a.tables[b * a.table_stride + r.old_pages + (j - page_pre[b])] = id;
    }
    // rows: positions and slots.  A request's pages before old_pages are in its table, the others
    // come from new_blocks (another thread writes them into the table).
    const int n_tokens = min(static_cast<int>(sum.rows), a.max_tokens);
    int64_t* meta_slots = reinterpret_cast<int64_t*>(a.meta + kHdrBytes);
    for (int i = me; i < n_tokens; i += stride) {
        const int b = last_at_most<uint32_t>(row_pre, B, i);
        const Request r = load_request(a, b);
        const uint32_t pos = r.ctx + (i - row_pre[b]);  // below 2^32
        int64_t slot = -1;
        if (served(a, r, row_pre[b], page_pre[b])) {
            const uint32_t page = pos / bs;
            const int32_t id = page < r.old_pages ? a.tables[b * a.table_stride + page]
                                                  : __ldg(a.new_blocks + page_pre[b] + (page - r.old_pages));
            if (static_cast<uint32_t>(id) < static_cast<uint32_t>(a.total_blocks))
                slot = static_cast<int64_t>(id) * bs + (pos - page * bs);
            else
                atomicOr(a.err, kErrBadBlock);
        }
        meta_slots[i] = slot;
        if (a.slots) a.slots[i] = slot;
        if (a.positions) a.positions[i] = static_cast<int32_t>(min(pos, 0x7fffffffu));
    }
}

__global__ void order_kernel() {}

}  // namespace

cudaError_t launch_step_build(const StepBuildArgs& a, cudaStream_t st) {
    if (a.batch < 0 || a.batch > kMaxBuildBatch) return cudaErrorInvalidValue;
    const int64_t n_seg = static_cast<int64_t>(a.batch) * a.heads_kv;
    if (a.n_workers < 1 || a.n_workers >= 1 << 14 || a.heads_kv >= 1 << 10 || n_seg >= 1 << 20) return cudaErrorInvalidValue;
    const size_t smem = static_cast<size_t>(a.batch + 1) * 8 + static_cast<size_t>(n_seg < kSegInSmem ? n_seg : kSegInSmem) * 8;
    if (smem > 40 * 1024) {  // above the default limit; set per device, cheap enough for so large a batch
        cudaError_t e = cudaFuncSetAttribute(step_build_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (kMaxBuildBatch + 1) * 8 + kSegInSmem * 8);
        if (e != cudaSuccess) return e;
    }
    // the merge entries and every 1024 workers; then a block for every 2048 rows or opened pages (4096: 8.5 us for 6.5 with 60000 rows)
    const int n_plan = 1 + (a.n_workers + kThreads - 1) / kThreads;
    const int64_t items = a.max_tokens > a.n_new_blocks ? a.max_tokens : a.n_new_blocks;
    int64_t fill = (items + 2 * kThreads - 1) / (2 * kThreads);
    fill = fill < 1 ? 1 : (fill > 128 ? 128 : fill);
    step_build_kernel<<<static_cast<unsigned>(n_plan + fill), kThreads, smem, st>>>(a, n_plan);
    return cudaGetLastError();
}

cudaError_t launch_order(cudaStream_t st) {
    order_kernel<<<1, 32, 0, st>>>();
    return cudaGetLastError();
}

}  // namespace gkv
