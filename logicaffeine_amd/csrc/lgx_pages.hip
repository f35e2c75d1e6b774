// lgx_pages.hip -- the pages of a paged cache: holders counted per page, sequences
// forked, pages reserved, copied and freed, all on the device.
//
// State: ref[page], the number of table entries that name the page (0: free), and the
// page table, -1 where an entry has no page.  Every result is a function of the
// inputs alone: counts are sums, and which page an entry gets is fixed by the order of
// entries and of free pages, not by the order of workgroups.
//
// All but the copy are a launch and a few dependent rounds: fork 2.4 to 4.1 us, free 1.8 to
// 4.0, reserve 3.4 for 2 sequences and 6.9 for 96 of 1728 pages.  The reserve is one
// workgroup because its order is the result: split over several it would have to pass the
// counts of needs and of free pages on, each a launch of its own.  The copy is bound by
// memory: 83 MB (45 pages in 56 planes, read and written) in 15.7 to 17.9 us, 4.6 to 5.3 TB/s.

#include "lgx_device.h"

// Exclusive sums over the workgroup's threads; total: of all.  sums: one per wave.
template <int NT>
__device__ __forceinline__ int block_scan(int v, int* sums, int& total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int upto = wave_scan(v);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    const int w = wave_scan(lane < NT / 64 ? sums[lane] : 0);
    total = __builtin_amdgcn_readlane(w, 63);
    const int before = wave ? __builtin_amdgcn_readlane(w, wave - 1) : 0;
    __syncthreads();
    return before + upto - v;
}

// Workgroup (pair, 256 entries of a row).  A pair whose rows are not both among the S,
// whose target is a source of the call, or is an earlier pair's target too, is left out:
// its row would be read and written at once.
extern "C" __global__ __launch_bounds__(256) void lgx_k_pages_fork(const lgx_fork_args a) {
    const int i = blockIdx.x, s = a.src[i], d = a.dst[i];
    bool out = s < 0 || s >= a.S || d < 0 || d >= a.S;
    for (int j = threadIdx.x; j < a.n; j += 256) out = out || a.src[j] == d || (j < i && a.dst[j] == d);
    if (__syncthreads_or(out)) return;
    const int len = min(max(a.seq_len[s], 0), a.maxp * LGX_PAGE), held = (len + LGX_PAGE - 1) / LGX_PAGE;
    const int col = blockIdx.y * 256 + threadIdx.x;
    if (col == 0) a.seq_len[d] = len;
    if (col >= a.maxp) return;
    int32_t* to = a.page_table + (int64_t)d * a.maxp + col;
    const int old = *to;
    int page = col < held ? a.page_table[(int64_t)s * a.maxp + col] : -1;
    if (page < 0 || page >= a.num_pages) page = -1;
    if (old >= 0 && old < a.num_pages) atomicSub(a.ref + old, 1);
    if (page >= 0) atomicAdd(a.ref + page, 1);
    *to = page;
}

extern "C" __global__ __launch_bounds__(256) void lgx_k_pages_free(const lgx_pages_free_args a) {
    const int b = blockIdx.x, col = blockIdx.y * 256 + threadIdx.x;
    const int64_t first = ((int64_t)max(a.keep[b], 0) + LGX_PAGE - 1) / LGX_PAGE;
    if (col >= a.maxp || col < first) return;
    int32_t* e = a.page_table + (int64_t)b * a.maxp + col;
    const int page = *e;
    if (page >= 0 && page < a.num_pages) atomicSub(a.ref + page, 1);
    if (page != -1) *e = -1;
}

// One workgroup, a thread per sequence: how many pages each needs, then as many free
// pages from the lowest up, then the entries in order of (sequence, entry).  Nothing is
// written unless all needs are met.  The free pages are found in rounds of 4 per thread
// until there are enough.
extern "C" __global__ __launch_bounds__(1024) void lgx_k_pages_reserve(const lgx_reserve_args a) {
    __shared__ int sums[16];
    __shared__ int page_s[LGX_PAGES_SEQS];        // the shared page that a sequence would write to, or -1
    const int b = threadIdx.x;
    const bool on = b < a.B;
    const int sl = on ? min(max(a.seq_len[b], 0), a.maxp * LGX_PAGE) : 0;
    const int need = on ? max(a.need[b], 0) : 0;
    const int first = sl / LGX_PAGE;
    const int end = (int)min(((int64_t)sl + need + LGX_PAGE - 1) / LGX_PAGE, (int64_t)a.maxp);
    int32_t* row = a.page_table + (int64_t)(on ? b : 0) * a.maxp;
    auto none = [&](int p) { return p < 0 || p >= a.num_pages; };
    int count = 0, page = -1, holders = 0;
    if (need > 0) {
        for (int e = first; e < end; ++e) count += none(row[e]);
        // tokens of the sequence stand in its entry `first`: only a copy of its own may be written
        if (sl % LGX_PAGE) {
            const int p = row[first];
            holders = none(p) ? 0 : a.ref[p];
            page = holders > 1 ? p : -1;
        }
    }
    page_s[b] = page;
    __syncthreads();
    // the last holder may keep the page: the others have left it
    int before = 0;
    if (page >= 0)
        for (int i = 0; i < b; ++i) before += page_s[i] == page;
    const bool leave = page >= 0 && before < holders - 1;
    int total, ncopy;
    int at = block_scan<1024>(count + leave, sums, total);
    const int copy = block_scan<1024>(leave, sums, ncopy);
    int got = 0;
    for (int64_t p0 = 0; p0 < a.num_pages && got < total; p0 += 4096) {   // uniform
        const int64_t p = p0 + 4 * b;
        bool f[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = p + i < a.num_pages && a.ref[min(p + i, (int64_t)a.num_pages - 1)] == 0;
            n += f[i];
        }
        int more, k = got + block_scan<1024>(n, sums, more);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (f[i] && k < total) a.found[k] = (int)(p + i);
            k += f[i];
        }
        got += more;
    }
    if (b == 0) {
        *a.lacking = max(total - got, 0);
        *a.n_copies = got < total ? 0 : ncopy;
    }
    if (got < total) return;                      // uniform
    __syncthreads();                              // the list is written
    if (leave) {
        const int p = a.found[at++];
        a.copies[2 * copy] = page;
        a.copies[2 * copy + 1] = p;
        row[first] = p;
        a.ref[p] = 1;
        atomicSub(a.ref + page, 1);
    }
    if (count > 0)
        for (int e = first; e < end; ++e)
            if (none(row[e])) {
                const int p = a.found[at++];
                row[e] = p;
                a.ref[p] = 1;
            }
}

// Workgroup (copy, plane): a page's bytes.
extern "C" __global__ __launch_bounds__(256) void lgx_k_pages_copy(const lgx_pages_copy_args a) {
    if ((int)blockIdx.x >= min(*a.n_copies, a.max)) return;
    const int s = a.copies[2 * blockIdx.x], d = a.copies[2 * blockIdx.x + 1];
    if (s < 0 || s >= a.num_pages || d < 0 || d >= a.num_pages || s == d) return;
    const int64_t n = a.bytes[blockIdx.y];
    char* base = a.base[blockIdx.y];
    const char* src = base + s * n;
    char* dst = base + d * n;
    if ((((uintptr_t)base | n) & 15) == 0) {
        for (int64_t i = threadIdx.x; i < n / 16; i += 256) ((uint4*)dst)[i] = ((const uint4*)src)[i];
    } else if ((((uintptr_t)base | n) & 3) == 0) {
        for (int64_t i = threadIdx.x; i < n / 4; i += 256) ((uint32_t*)dst)[i] = ((const uint32_t*)src)[i];
    } else {
        for (int64_t i = threadIdx.x; i < n; i += 256) dst[i] = src[i];
    }
}
