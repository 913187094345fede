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
// wait between its blocks: each block repeats the scan over the requests (at most 4096, from L2),
// block 0 plans, the others write tables, slots and positions.
#include "gkv_device.cuh"
#include "kernels.h"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Exclusive prefix of x over the block; total gets the sum.  One call may follow another.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* warp_sum, int64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();  // the last call's reads of warp_sum are done
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    const int64_t mine = lane < kWarps ? warp_sum[lane] : 0;
    int64_t s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, s, o);
        if (lane >= o) s += y;
    }
    total = __shfl_sync(~0u, s, 31);
    return __shfl_sync(~0u, s - mine, warp) + inc - x;
}

// floor(a / b) for 0 <= a < 2^62, b > 0 and a quotient below 2^51: a rounded estimate, put right by
// products (a 64-bit division is some hundred cycles).
__device__ __forceinline__ int64_t floor_div(int64_t a, int64_t b, double inv_b) {
    int64_t q = static_cast<int64_t>(static_cast<double>(a) * inv_b);
    while (q > 0 && q * b > a) --q;
    while ((q + 1) * b <= a) ++q;
    return q;
}

__device__ __forceinline__ int64_t chunks_in(int64_t ctx, int bs) {
    const int64_t cpp = (bs + kDecodeChunk - 1) / kDecodeChunk;
    const int64_t full = ctx / bs;
    return full * cpp + (ctx - full * bs + kDecodeChunk - 1) / kDecodeChunk;
}

struct Request {
    int64_t ctx, n;   // as given, negative ones as 0
    int64_t old_pages, opened;
    bool fits;        // lengths valid and within the table row
};

__device__ __forceinline__ Request load_request(const StepBuildArgs& a, int b) {
    Request r;
    const int c = __ldg(a.ctx_lens + b), n = __ldg(a.new_lens + b);
    r.ctx = c > 0 ? c : 0;
    r.n = n > 0 ? n : 0;
    const int64_t end = r.ctx + r.n;
    r.fits = c >= 0 && n >= 0 && end <= 0x7fffffff && end <= a.table_stride * a.block_size;
    r.old_pages = (r.ctx + a.block_size - 1) / a.block_size;
    r.opened = r.fits ? (end + a.block_size - 1) / a.block_size - r.old_pages : 0;
    return r;
}

__device__ __forceinline__ int saturate(int64_t x) { return x > 0x7fffffff ? 0x7fffffff : static_cast<int>(x); }

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

__device__ __forceinline__ bool served(const StepBuildArgs& a, const Request& r, int64_t row0, int64_t page0) {
    return r.fits && (r.n == 0 || row0 + r.n <= a.max_tokens) && (r.opened == 0 || page0 + r.opened <= a.n_new_blocks);
}

// ---- the work list ------------------------------------------------------------------------

// The stream of units, as the planning block holds it: segment (b, h) spans units
// [pre[b] * H + h * span, ... + span), span = pre[b + 1] - pre[b] = kSegmentCost + its chunks, or 0.
struct Units {
    const int64_t* pre;   // [batch + 1], one head's units
    const int32_t* live;  // [batch + 1], requests with units before b
    int batch, H;
    int64_t total, n;     // units in all, workers
    double inv_total, inv_n;

    // first unit of worker w
    __device__ __forceinline__ int64_t begin(int64_t w) const { return floor_div(w * total, n, inv_n); }
    // the worker that holds unit u
    __device__ __forceinline__ int64_t worker_of(int64_t u) const {
        return floor_div((u + 1) * n - 1, total, inv_total);  // = ceil((u + 1) n / total) - 1
    }
    // segment of unit u: request and head
    __device__ __forceinline__ void segment_of(int64_t u, int& b, int& h) const {
        const int64_t per_head = u / H;  // pre[b] <= u / H < pre[b + 1]
        b = last_at_most<int64_t>(pre, batch, per_head);
        const int64_t span = pre[b + 1] - pre[b];
        h = static_cast<int>((u - pre[b] * H) / span);
    }
};

__device__ void plan(const StepBuildArgs& a, const Units& U, int64_t* warp_sum, int n_tokens) {
    int32_t* pseg = reinterpret_cast<int32_t*>(a.meta + a.off_pseg);
    int32_t* pc0 = reinterpret_cast<int32_t*>(a.meta + a.off_pc0);
    int32_t* pc1 = reinterpret_cast<int32_t*>(a.meta + a.off_pc1);
    int32_t* pslot = reinterpret_cast<int32_t*>(a.meta + a.off_pslot);
    int32_t* pmerge = reinterpret_cast<int32_t*>(a.meta + a.off_pmerge);
    int32_t* wbeg = reinterpret_cast<int32_t*>(a.meta + a.off_wbeg);
    int32_t* mseg = reinterpret_cast<int32_t*>(a.meta + a.off_mseg);
    int32_t* ms0 = reinterpret_cast<int32_t*>(a.meta + a.off_ms0);
    int32_t* mns = reinterpret_cast<int32_t*>(a.meta + a.off_mns);
    int32_t* mdef = reinterpret_cast<int32_t*>(a.meta + a.off_mdef);
    const int H = U.H;
    const int n_seg = U.batch * H;
    int32_t* seg_slot = a.scratch;          // [n_seg] first partial slot, -1 for a segment in one piece
    int32_t* long_before = a.scratch + n_seg;  // [n_merge]

    // segments: their pieces, partial slots and merge entries
    int64_t merges = 0, slots = 0, longs = 0;
    for (int base = 0; base < n_seg; base += kThreads) {
        const int s = base + static_cast<int>(threadIdx.x);
        int64_t pieces = 0;
        if (s < n_seg) {
            const int b = s / H, h = s - b * H;
            const int64_t span = U.pre[b + 1] - U.pre[b];
            if (span > 0) {
                const int64_t s0 = U.pre[b] * H + h * span;
                // workers with units in [s0 + cost, s0 + span); one unit each when units are fewer than workers
                pieces = U.total >= U.n ? U.worker_of(s0 + span - 1) - U.worker_of(s0 + kSegmentCost) + 1 : span - kSegmentCost;
            }
        }
        const bool split = pieces > 1;
        const bool is_long = pieces > kWarpMergeMaxSlots;
        // three counts in one scan: merge entries, long ones, slots (pieces are below 2^31 in all)
        int64_t tm, tls;
        const int64_t at_m = merges + block_scan(split, warp_sum, tm);
        const int64_t both = block_scan(split ? (pieces | (is_long ? int64_t{1} << 40 : 0)) : 0, warp_sum, tls);
        const int64_t at_s = slots + (both & ((int64_t{1} << 40) - 1));
        const int64_t at_l = longs + (both >> 40);
        if (s < n_seg) seg_slot[s] = split ? static_cast<int32_t>(at_s) : -1;
        if (split) {
            mseg[at_m] = s;
            ms0[at_m] = static_cast<int32_t>(at_s);
            mns[at_m] = static_cast<int32_t>(pieces);
            long_before[at_m] = static_cast<int32_t>(at_l);
        }
        merges += tm;
        slots += tls & ((int64_t{1} << 40) - 1);
        longs += tls >> 40;
    }
    __syncthreads();
    // the deferred list: every split segment, the long ones first, each kind in order
    static_assert(kFusedMergeMaxSlots == 0, "the list below defers every merge");
    for (int m = static_cast<int>(threadIdx.x); m < merges; m += kThreads) {
        const int lb = long_before[m];
        mdef[mns[m] > kWarpMergeMaxSlots ? lb : longs + m - lb] = m;
    }

    // workers: number their pieces, then write them
    int64_t pieces_before = 0;
    const int n_workers = a.n_workers;
    for (int base = 0; base < n_workers; base += kThreads) {
        const int w = base + static_cast<int>(threadIdx.x);
        int64_t lo = 0, hi = 0;
        int b = 0, h = 0;
        int64_t count = 0;
        if (w < n_workers && U.total > 0) {
            lo = U.begin(w);
            hi = U.begin(w + 1);
            if (lo < hi) {
                int b1, h1;
                U.segment_of(lo, b, h);
                U.segment_of(hi - 1, b1, h1);
                // live segments from the first to the last; the last has no piece when the range ends inside its overhead
                count = static_cast<int64_t>(U.live[b1] - U.live[b]) * H + (h1 - h) + 1;
                const int64_t span = U.pre[b1 + 1] - U.pre[b1];
                if (hi <= U.pre[b1] * H + h1 * span + kSegmentCost) --count;
            }
        }
        int64_t total;
        const int64_t at = pieces_before + block_scan(count, warp_sum, total);
        if (w < n_workers) wbeg[w] = static_cast<int32_t>(at);
        for (int64_t k = at; k < at + count; ++k) {
            const int64_t span = U.pre[b + 1] - U.pre[b];
            const int64_t s0 = U.pre[b] * H + h * span;
            const int seg = b * H + h;
            const int64_t c0 = max(lo - s0 - kSegmentCost, int64_t{0});
            const int64_t c1 = min(hi, s0 + span) - s0 - kSegmentCost;
            const int first = seg_slot[seg];
            pseg[k] = seg;
            pc0[k] = static_cast<int32_t>(c0);
            pc1[k] = static_cast<int32_t>(c1);
            // pieces of a segment are consecutive workers', or single units
            pslot[k] = first < 0 ? -1 : first + static_cast<int32_t>(U.total >= U.n ? w - U.worker_of(s0 + kSegmentCost) : c0);
            pmerge[k] = first < 0 ? -1 : -2;
            if (k + 1 < at + count && ++h == H) {  // the next live segment
                h = 0;
                do ++b;
                while (U.pre[b + 1] == U.pre[b]);
            }
        }
        pieces_before += total;
    }
    if (threadIdx.x == 0) {
        wbeg[n_workers] = static_cast<int32_t>(pieces_before);
        int32_t* hd = reinterpret_cast<int32_t*>(a.meta);
        hd[kHdrTok] = n_tokens;
        hd[kHdrBatch] = a.batch;
        hd[kHdrMaxBlocks] = saturate(a.table_stride);
        hd[kHdrSlots] = static_cast<int32_t>(slots);
        hd[kHdrMerge] = static_cast<int32_t>(merges);
        hd[kHdrDeferred] = static_cast<int32_t>(merges);
        hd[kHdrDeferredLong] = static_cast<int32_t>(longs);
        hd[kHdrWorkers] = n_workers;
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
}

__global__ void __launch_bounds__(kThreads) step_build_kernel(const StepBuildArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int64_t warp_sum[kWarps];
    __shared__ int used_blocks, left_out;
    const int B = a.batch;
    const bool planner = blockIdx.x == 0;
    // exclusive prefixes over the requests: rows and opened pages (saturated: larger ones are never
    // searched for), and for the planner units and live requests
    int64_t* unit_pre = reinterpret_cast<int64_t*>(smem);
    int32_t* row_pre = planner ? reinterpret_cast<int32_t*>(unit_pre + B + 1) : reinterpret_cast<int32_t*>(smem);
    int32_t* page_pre = row_pre + B + 1;
    int32_t* live_pre = page_pre;  // the planner's
    if (threadIdx.x == 0) used_blocks = left_out = 0;
    __syncthreads();

    int64_t rows = 0, pages = 0, units = 0, live = 0;
    for (int base = 0; base < B; base += kThreads) {
        const int b = base + static_cast<int>(threadIdx.x);
        Request r{};
        if (b < B) r = load_request(a, b);
        int64_t tr, tp;
        const int64_t row0 = rows + block_scan(r.n, warp_sum, tr);
        const int64_t page0 = pages + block_scan(r.opened, warp_sum, tp);
        rows += tr;
        pages += tp;
        const bool ok = b < B && served(a, r, row0, page0);
        if (planner) {
            const int64_t ctx = ok ? r.ctx + r.n : 0;
            const int64_t c = chunks_in(ctx, a.block_size);
            int64_t tu, tl;
            const int64_t unit0 = units + block_scan(c > 0 ? c + kSegmentCost : 0, warp_sum, tu);
            const int64_t live0 = live + block_scan(c > 0, warp_sum, tl);
            units += tu;
            live += tl;
            if (b < B) {
                unit_pre[b] = unit0;
                live_pre[b] = static_cast<int32_t>(live0);
                reinterpret_cast<int32_t*>(a.meta + a.off_ctx)[b] = static_cast<int32_t>(ctx);
            }
        } else if (b < B) {
            row_pre[b] = saturate(row0);
            page_pre[b] = saturate(page0);
            if (blockIdx.x == 1) {  // this block also writes what there is one of per request
                if (a.cu_new) a.cu_new[b] = saturate(row0);
                if (a.ctx_out) a.ctx_out[b] = static_cast<int32_t>(ok ? r.ctx + r.n : r.ctx);
                if (ok && r.opened > 0) atomicMax(&used_blocks, static_cast<int>(page0 + r.opened));
                if (!ok) left_out = 1;
            }
        }
    }
    const int n_tokens = rows < a.max_tokens ? static_cast<int>(rows) : a.max_tokens;
    if (threadIdx.x == 0) {
        if (planner) {
            unit_pre[B] = units;
            live_pre[B] = static_cast<int32_t>(live);
        } else {
            row_pre[B] = saturate(rows);
            page_pre[B] = saturate(pages);
        }
    }
    __syncthreads();

    if (planner) {
        const int64_t total = units * a.heads_kv;
        const Units U{unit_pre, live_pre, B, a.heads_kv, total, a.n_workers, 1.0 / static_cast<double>(total > 0 ? total : 1),
                      1.0 / static_cast<double>(a.n_workers)};
        plan(a, U, warp_sum, n_tokens);
        return;
    }
    if (blockIdx.x == 1 && threadIdx.x == 0) {
        if (a.cu_new) a.cu_new[B] = saturate(rows);
        if (a.counts) {
            a.counts[0] = saturate(rows);
            a.counts[1] = used_blocks;
        }
        if (left_out) atomicOr(a.err, kErrBadStep);
    }

    const int bs = a.block_size;
    const int stride = static_cast<int>((gridDim.x - 1) * kThreads);
    const int me = static_cast<int>((blockIdx.x - 1) * kThreads + threadIdx.x);
    // opened pages into the tables
    const int n_pages = pages < a.n_new_blocks ? static_cast<int>(pages) : a.n_new_blocks;
    for (int j = me; j < n_pages; j += stride) {
        const int b = last_at_most<int32_t>(page_pre, B, j);
        const Request r = load_request(a, b);
        if (!served(a, r, row_pre[b], page_pre[b])) continue;
        const int32_t id = __ldg(a.new_blocks + j);
        if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.total_blocks)) atomicOr(a.err, kErrBadBlock);
        a.tables[b * a.table_stride + r.old_pages + (j - page_pre[b])] = id;
    }
    // rows: positions and slots.  A request's pages before old_pages are in its table, the others
    // come from new_blocks (another thread writes them into the table).
    int64_t* meta_slots = reinterpret_cast<int64_t*>(a.meta + kHdrBytes);
    for (int i = me; i < n_tokens; i += stride) {
        const int b = last_at_most<int32_t>(row_pre, B, i);
        const Request r = load_request(a, b);
        const int64_t pos = r.ctx + (i - row_pre[b]);
        int64_t slot = -1;
        if (served(a, r, row_pre[b], page_pre[b])) {
            const int page = static_cast<int>(pos) / bs;
            const int32_t id = page < r.old_pages ? a.tables[b * a.table_stride + page]
                                                  : __ldg(a.new_blocks + page_pre[b] + (page - static_cast<int>(r.old_pages)));
            if (static_cast<uint32_t>(id) < static_cast<uint32_t>(a.total_blocks))
                slot = static_cast<int64_t>(id) * bs + (static_cast<int>(pos) - page * bs);
            else
                atomicOr(a.err, kErrBadBlock);
        }
        meta_slots[i] = slot;
        if (a.slots) a.slots[i] = slot;
        if (a.positions) a.positions[i] = saturate(pos);
    }
}

__global__ void order_kernel() {}

}  // namespace

cudaError_t launch_step_build(const StepBuildArgs& a, cudaStream_t st) {
    if (a.batch < 0 || a.batch > kMaxBuildBatch) return cudaErrorInvalidValue;
    const size_t smem = static_cast<size_t>(a.batch + 1) * 16;
    if (smem > 40 * 1024) {  // above the default limit; set per device, cheap enough for so large a batch
        cudaError_t e = cudaFuncSetAttribute(step_build_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxBuildBatch + 1) * 16);
        if (e != cudaSuccess) return e;
    }
    // the planner, and a block for every 4096 rows or opened pages
    const int64_t items = a.max_tokens > a.n_new_blocks ? a.max_tokens : a.n_new_blocks;
    int64_t fill = (items + 4 * kThreads - 1) / (4 * kThreads);
    fill = fill < 1 ? 1 : (fill > 147 ? 147 : fill);
    step_build_kernel<<<static_cast<unsigned>(1 + fill), kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_order(cudaStream_t st) {
    order_kernel<<<1, 32, 0, st>>>();
    return cudaGetLastError();
}

}  // namespace gkv
