// Block tables and slot maps from request lengths, in one launch (formulas: pocket_tts_amd.h, ptts_paged_plan).
//
// Every workgroup scans all request lengths itself, a chunk of requests at a time, and keeps only the exclusive prefix sums of one
// chunk in LDS; it then writes the packed rows of its own slice of the rows and the table entries of its own slice of the
// picked pages that fall into the chunk.  One launch and no order between workgroups: nobody reads a table entry that the
// call writes, because whether a page is old (table) or new (free list) follows from the lengths alone.
//
// The sizes are small and the time is a chain of latencies (arguments, lengths, a table entry, the stores), so the chain is kept
// short: the one old table entry that a request's new rows can fall into is read while the sums are formed, and the head of the
// free list is read at the start.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "paged.h"

namespace ptts {

namespace {

constexpr int kSlice = 256;           // packed rows, and picked pages, of one workgroup

struct PlanArgs {
    PttsPagedPlan p;
    FastDiv page;
    long long picks;                  // picked pages dealt out in slices; the last workgroup takes whatever lies beyond
};

__device__ __forceinline__ long long wave_scan_incl(long long v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
    }
    return v;
}

// index of the last entry of a[0 .. n] (ascending, a[0] <= x < a[n]) that is <= x
__device__ __forceinline__ int find_last(const long long* a, int n, long long x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// kPer requests a thread and chunk: 1 for up to 256 requests (one round of loads; 64 requests 4.5 us, with 4 a thread 5.4), 4 above (fewer
// rounds of sums; 509 requests with 130 thousand rows 6.3 us, with 1 a thread 6.4).  An empty launch takes about 4.
template <int kPer> __global__ __launch_bounds__(256) void plan_kernel(PlanArgs a) {
    constexpr int kChunk = 256 * kPer;
    __shared__ long long row0[kChunk + 1], pick0[kChunk + 1];
    __shared__ int cached[kChunk], have[kChunk], tail[kChunk], head[256];
    __shared__ long long part[2][4];
    const PttsPagedPlan& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ps = p.page_size;
    const bool last_wg = blockIdx.x + 1 == gridDim.x;
    const long long r_lo = (long long)blockIdx.x * kSlice, r_hi = r_lo + kSlice < p.rows ? r_lo + kSlice : p.rows;
    const long long k_lo = (long long)blockIdx.x * kSlice, k_hi = last_wg ? (1ll << 62) : k_lo + kSlice;
    long long rows_before = 0, picks_before = 0, lost_pages = 0, no_page = 0;
    int bad = 0;
    head[tid] = tid < p.n_free ? p.free_pages[tid] : -1;
    auto free_page = [&](long long pick) { return pick < 256 ? head[pick] : pick < p.n_free ? p.free_pages[pick] : -1; };
    for (int c0 = 0; c0 < p.requests; c0 += kChunk) {
        const int n = p.requests - c0 < kChunk ? p.requests - c0 : kChunk;
        const int i0 = kPer * tid;
        int cach[kPer], arr[kPer], hv[kPer], need[kPer], old[kPer];
        long long rs = 0, ks = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            cach[j] = arr[j] = 0;
            if (i0 + j < n) {
                cach[j] = p.cached[c0 + i0 + j];
                arr[j] = p.arriving[c0 + i0 + j];
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (cach[j] < 0) { cach[j] = 0; bad = 1; }
            if (arr[j] < 0) { arr[j] = 0; bad = 1; }
            if (arr[j] > 0x7fffffff - cach[j]) { arr[j] = 0; bad = 1; }
            const int end = cach[j] + arr[j], full = (int)a.page.div(cach[j]);
            int h = full, e = (int)a.page.div(end);
            h += h * ps < cach[j];
            e += (long long)e * ps < end;
            if (h > p.table_width) { h = p.table_width; bad = 1; }
            // new rows meet one old page at most: the last one, where it is partly filled
            old[j] = full < h && arr[j] > 0 ? p.block_table[(long long)(c0 + i0 + j) * p.table_stride + full] : -1;
            const int fit = e < p.table_width ? e : p.table_width;
            lost_pages += e - (fit > h ? fit : h);
            hv[j] = h;
            need[j] = fit > h ? fit - h : 0;
            rs += arr[j];
            ks += need[j];
        }
        const long long ri = wave_scan_incl(rs), ki = wave_scan_incl(ks);
        __syncthreads();                       // the previous chunk's prefix sums are no longer read
        if (lane == 63) { part[0][wave] = ri; part[1][wave] = ki; }
        __syncthreads();
        long long r = rows_before + ri - rs, k = picks_before + ki - ks;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) { r += part[0][w]; k += part[1][w]; }
            rows_before += part[0][w];
            picks_before += part[1][w];
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            row0[i0 + j] = r;
            pick0[i0 + j] = k;
            cached[i0 + j] = cach[j];
            have[i0 + j] = hv[j];
            tail[i0 + j] = old[j];
            if (i0 + j < n && (unsigned)(c0 / kChunk) % gridDim.x == blockIdx.x) {
                p.cu_rows[c0 + i0 + j] = (int)(r < 0x7fffffff ? r : 0x7fffffff);
                p.kv_len[c0 + i0 + j] = cach[j] + arr[j];
            }
            // rows of this request that end up without a page: those of a held page that is missing (an earlier plan's -1), and those
            // behind the last page that it holds or gets
            const int full = (int)a.page.div(cach[j]);
            if (full < hv[j] && arr[j] > 0 && old[j] < 0) {
                const long long room = (full + 1ll) * ps - cach[j];
                no_page += arr[j] < room ? arr[j] : room;
            }
            const long long got = p.n_free - k < 0 ? 0 : p.n_free - k < need[j] ? p.n_free - k : need[j];
            const long long first_out = (hv[j] + got) * ps > cach[j] ? (hv[j] + got) * ps : cach[j];
            if (cach[j] + (long long)arr[j] > first_out) no_page += cach[j] + (long long)arr[j] - first_out;
            r += arr[j];
            k += need[j];
        }
        if (tid == 255) { row0[kChunk] = r; pick0[kChunk] = k; }
        __syncthreads();
        // packed rows of this workgroup's slice
        const long long ra = r_lo > row0[0] ? r_lo : row0[0], rb = r_hi < row0[n] ? r_hi : row0[n];
        for (long long q = ra + tid; q < rb; q += 256) {
            const int i = find_last(row0, n, q), pos = cached[i] + (int)(q - row0[i]), pg = (int)a.page.div(pos);
            int id = -1;
            if (pg < p.table_width) id = pg < have[i] ? tail[i] : free_page(pick0[i] + pg - have[i]);
            long long slot = id < 0 ? -1 : (long long)id * ps + (pos - pg * ps);
            if (slot > 0x7fffffff) { slot = -1; bad |= 2; }
            p.slot_map[q] = (int)slot;
            p.positions[q] = pos;
        }
        // table entries of this workgroup's slice of the picked pages
        const long long ka = k_lo > pick0[0] ? k_lo : pick0[0], kb = k_hi < pick0[n] ? k_hi : pick0[n];
        for (long long q = ka + tid; q < kb; q += 256) {
            const int i = find_last(pick0, n, q);
            const int id = free_page(q);
            if (id < 0 && q < p.n_free) bad |= 2;
            p.block_table[(long long)(c0 + i) * p.table_stride + have[i] + (int)(q - pick0[i])] = id;
        }
    }
    // totals, the same in every workgroup
    if (blockIdx.x == 0) {
        __syncthreads();
        long long lp = lost_pages, np = no_page;
        for (int o = 32; o > 0; o >>= 1) { lp += __shfl_xor(lp, o, 64); np += __shfl_xor(np, o, 64); }
        if (lane == 0) { part[0][wave] = lp; part[1][wave] = np; }
        __syncthreads();
        if (tid == 0) {
            lp = part[0][0] + part[0][1] + part[0][2] + part[0][3];
            np = part[1][0] + part[1][1] + part[1][2] + part[1][3];
            const long long taken = picks_before < p.n_free ? picks_before : p.n_free;
            const long long missing = picks_before - taken + lp;
            p.cu_rows[p.requests] = (int)(rows_before < 0x7fffffff ? rows_before : 0x7fffffff);
            p.counts[0] = p.cu_rows[p.requests];
            p.counts[1] = (int)taken;
            p.counts[2] = (int)(missing < 0x7fffffff ? missing : 0x7fffffff);
            p.counts[3] = (int)(np < 0x7fffffff ? np : 0x7fffffff);
        }
    }
    if (p.status && bad) atomicOr(p.status, ((bad & 1) ? kStatusLength : 0) | ((bad & 2) ? kStatusPage : 0));
}

}  // namespace

void check_paged_plan(const PttsPagedPlan& p) {
    if (p.requests < 0 || p.requests > 65536) throw std::runtime_error("requests must be 0 to 65536");
    if (p.page_size < 1 || p.page_size >= 1 << 30) throw std::runtime_error("page_size must be 1 to 2^30 - 1");
    if (p.table_width < 0 || p.n_free < 0 || p.rows < 0) throw std::runtime_error("table_width, n_free and rows must not be negative");
    if (p.requests > 1 && p.table_stride < p.table_width) throw std::runtime_error("table_stride is smaller than table_width");
    if (p.requests > 0 && (!p.cached || !p.arriving || !p.kv_len || (p.table_width > 0 && !p.block_table)))
        throw std::runtime_error("cached, arriving, kv_len and block_table are required");
    if (!p.cu_rows || !p.counts) throw std::runtime_error("cu_rows and counts are required");
    if (p.rows > 0 && (!p.slot_map || !p.positions)) throw std::runtime_error("slot_map and positions are required");
    if (!aligned({p.cached, p.arriving, p.free_pages, p.block_table, p.slot_map, p.positions, p.cu_rows, p.kv_len, p.counts, p.status}, 4))
        throw std::runtime_error("all arrays must be aligned to 4 bytes");
    if (p.n_free > 0 && !p.free_pages) throw std::runtime_error("free_pages is required");
}

void launch_paged_plan(const PttsPagedPlan& p, hipStream_t s) {
    PlanArgs a;
    a.p = p;
    a.page = FastDiv::of(static_cast<unsigned>(p.page_size));
    // lengths that fit `rows` never pick more pages than this
    const long long most = static_cast<long long>(p.rows) / p.page_size + p.requests;
    a.picks = most < p.n_free ? most : p.n_free;
    const long long slices = std::max<long long>((p.rows + kSlice - 1) / kSlice, (a.picks + kSlice - 1) / kSlice);
    const dim3 grid(static_cast<unsigned>(std::max<long long>(slices, 1)));
    if (p.requests <= 256) launch_paged(plan_kernel<1>, grid, s, a);
    else launch_paged(plan_kernel<4>, grid, s, a);
}

}  // namespace ptts
