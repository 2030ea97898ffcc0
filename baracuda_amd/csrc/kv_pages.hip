// kv_pages.hip -- pages of a key-value cache: copy, fork, release, compact.
//
// The cache is [layers, pages, page bytes]; one page table serves all layers.
// tables [rows, max_pages] holds a sequence's pages in order (-1: none), lens
// its tokens, refs how many rows hold a page.  Everything is decided on the
// device from these, so a captured graph replays with whatever they hold then.
//
// The moves themselves are a copy: bound by HBM, one read and one write of each
// moved byte.  What decides about them is a scan over the pages by one
// workgroup, in whole numbers, so that the lowest free page is taken first
// whatever order the waves run in.  Measured: 7 pages of 17 KiB in 32 layers copied
// in 4.1 us; 16 forks of two prompts, 2.2 MiB each, in 4.9 (the scan) and 12 us; 1200
// pages compacted, 267 of 34 KiB in 32 layers moved, in 6.5 and 103 us (5.7 TB/s; a
// large copy by the library 4.8).
#include "bk_common.hpp"

namespace bk {
namespace {

constexpr int kScan = 1024;

// Exclusive sum over the workgroup of kScan threads; `total` is the sum.
__device__ __forceinline__ int block_scan(int x, int *lds, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kScan / 64; ++w) {
        const int v = lds[w];
        before += w < wave ? v : 0;
        total += v;
    }
    return before + s - x;
}

// `bytes` from src to dst by the threads of the workgroup; V the unit.  STREAM:
// streaming loads and stores, for pages that nobody reads again soon: 267 pages of
// 34 KiB in 32 layers take 104 us with both hints (5.7 TB/s), 120 without.  Forks,
// which read one page many times, take 11.5 us without and 16.3 with them.
template <typename V, bool STREAM>
__device__ __forceinline__ void copy_span(uint8_t *__restrict__ dst, const uint8_t *__restrict__ src, int64_t bytes) {
    constexpr int U = 4;
    const int64_t n = bytes / (int64_t)sizeof(V), step = blockDim.x;
    const V *s = (const V *)src;
    V *d = (V *)dst;
    const auto get = [&](int64_t i) { return STREAM ? __builtin_nontemporal_load(&s[i]) : s[i]; };
    const auto put = [&](int64_t i, const V &v) {
        if (STREAM) __builtin_nontemporal_store(v, &d[i]);
        else d[i] = v;
    };
    int64_t i = threadIdx.x;
    for (; i + (U - 1) * step < n; i += U * step) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = get(i + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) put(i + u * step, v[u]);
    }
    for (; i < n; i += step) put(i, get(i));
}

// The moves of all layers, cut into spans; a workgroup takes every
// gridDim.x-th span.  moves: pairs of pages, `count` of them on the device or
// the host.
template <typename V, bool STREAM>
__device__ __forceinline__ void move_pages(uint8_t *cache, const int32_t *src, const int32_t *dst, int64_t count, int layers,
                                           int64_t pages, int64_t page_bytes, int64_t span, int64_t first, int64_t step) {
    const int64_t spans = (page_bytes + span - 1) / span;
    const int64_t total = count * layers * spans;
    for (int64_t u = first; u < total; u += step) {
        const int64_t part = u % spans, rest = u / spans;
        const int64_t m = rest % count, layer = rest / count;
        const int64_t from = src[m], to = dst[m];
        if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) continue;
        const int64_t at = part * span, bytes = page_bytes - at < span ? page_bytes - at : span;
        copy_span<V, STREAM>(cache + (layer * pages + to) * page_bytes + at, cache + (layer * pages + from) * page_bytes + at,
                             bytes);
    }
}

template <typename V>
__global__ __launch_bounds__(256) void copy_kernel(uint8_t *cache, const int32_t *src, const int32_t *dst, int64_t count,
                                                   int layers, int64_t pages, int64_t page_bytes, int64_t span) {
    move_pages<V, false>(cache, src, dst, count, layers, pages, page_bytes, span, blockIdx.x, gridDim.x);
}

// The page that each child gets for its parent's partly filled one: the lowest
// free pages, in the order of the children.  -1: it needs none; -2: there is
// none, or its parent or its own row is no row.
__global__ __launch_bounds__(kScan) void fork_plan_kernel(const int32_t *__restrict__ lens, const int32_t *__restrict__ refs,
                                                          const int32_t *__restrict__ parents,
                                                          const int32_t *__restrict__ children, int32_t *fresh, int n,
                                                          int rows, int pages, int ps, int max_pages) {
    __shared__ int lds[kScan / 64];
    const auto needs = [&](int i) {
        const int p = parents[i], c = children[i];
        if ((unsigned)p >= (unsigned)rows || (unsigned)c >= (unsigned)rows) return -1;
        const int len = lens[p];
        return len > 0 && len % ps != 0 && len / ps < max_pages ? 1 : 0;
    };
    int need = 0, total;
    for (int c0 = 0; c0 < n; c0 += kScan) {
        const int i = c0 + (int)threadIdx.x;
        (void)block_scan(i < n && needs(i) > 0, lds, total);
        need += total;
    }
    // the free pages in order, as a list in fresh[0..need)
    int found = 0;
    for (int p0 = 0; p0 < pages && found < need; p0 += kScan) {
        const int p = p0 + (int)threadIdx.x;
        const bool free = p < pages && refs[p] == 0;
        const int at = found + block_scan(free, lds, total);
        if (free && at < need) fresh[at] = p;
        found += total;
    }
    __syncthreads();
    __threadfence_block();
    // ... handed out from the last children back: a child's place in the list
    // is never behind its own, so what is read is not yet overwritten
    int after = need;
    for (int c0 = (n - 1) / kScan * kScan; c0 >= 0; c0 -= kScan) {
        const int i = c0 + (int)threadIdx.x;
        const int want = i < n ? needs(i) : 0;
        const int before = block_scan(want > 0, lds, total);
        after -= total;
        int page = want < 0 ? -2 : -1;
        if (want > 0) page = after + before < found ? fresh[after + before] : -2;
        __syncthreads();
        if (i < n) fresh[i] = page;
    }
}

// Tables, lengths and references of the children (the first n workgroups),
// then the copies of the partly filled pages.
template <typename V>
__global__ __launch_bounds__(256) void fork_kernel(uint8_t *cache, int32_t *tables, int32_t *lens, int32_t *refs,
                                                   const int32_t *__restrict__ parents, const int32_t *__restrict__ children,
                                                   const int32_t *__restrict__ fresh, int n, int rows, int max_pages,
                                                   int ps, int layers, int64_t pages, int64_t page_bytes, int64_t span) {
    if ((int)blockIdx.x < n) {
        const int i = blockIdx.x, p = parents[i], c = children[i], f = fresh[i];
        if ((unsigned)c >= (unsigned)rows) return;
        const bool lost = f < -1 || (unsigned)p >= (unsigned)rows;
        const int len = lost ? 0 : max(lens[p], 0), full = min(len / ps, max_pages);
        for (int j = threadIdx.x; j < max_pages; j += blockDim.x) {
            int e = -1;
            if (j < full) {
                e = tables[(int64_t)p * max_pages + j];
                if (e >= 0 && e < pages) atomicAdd(&refs[e], 1);
            } else if (j == full && f >= 0) {
                e = f;
                atomicAdd(&refs[f], 1);
            }
            tables[(int64_t)c * max_pages + j] = e;
        }
        if (threadIdx.x == 0) lens[c] = len;
        return;
    }
    const int64_t spans = (page_bytes + span - 1) / span;
    const int64_t total = (int64_t)n * layers * spans;
    for (int64_t u = (int64_t)blockIdx.x - n; u < total; u += (int64_t)gridDim.x - n) {
        const int64_t part = u % spans, rest = u / spans;
        const int i = (int)(rest % n);
        const int64_t layer = rest / n;
        const int to = fresh[i];
        if (to < 0) continue;
        // the parent's length is read again: should it be a child too, against what is
        // asked of the caller, it may be another one by now, as long as the table
        const int p = parents[i], last = lens[p] / ps;
        if (last >= max_pages) continue;
        const int from = tables[(int64_t)p * max_pages + last];
        if (from < 0 || from >= pages) continue;
        const int64_t at = part * span, bytes = page_bytes - at < span ? page_bytes - at : span;
        copy_span<V, false>(cache + (layer * pages + to) * page_bytes + at, cache + (layer * pages + from) * page_bytes + at, bytes);
    }
}

// A row named twice gives its pages back once: the exchange hands each entry to one thread.
__global__ __launch_bounds__(256) void release_kernel(int32_t *tables, int32_t *lens, int32_t *refs,
                                                      const int32_t *__restrict__ which, int rows, int max_pages, int pages) {
    const int r = which[blockIdx.x];
    if ((unsigned)r >= (unsigned)rows) return;
    for (int j = blockIdx.y * blockDim.x + threadIdx.x; j < max_pages; j += gridDim.y * blockDim.x) {
        const int e = atomicExch(&tables[(int64_t)r * max_pages + j], -1);
        if (e >= 0 && e < pages) atomicSub(&refs[e], 1);
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) lens[r] = 0;
}

// Pages in use past the first `live` go, lowest first, into the free ones
// before it.  plan: the number of moves, their sources, their destinations.
__global__ __launch_bounds__(kScan) void compact_plan_kernel(const int32_t *__restrict__ refs, int32_t *refs_out,
                                                             int32_t *remap, int32_t *live, int32_t *plan, int pages) {
    __shared__ int lds[kScan / 64];
    int32_t *src = plan + 4, *dst = src + pages;
    int count = 0, total;
    for (int p0 = 0; p0 < pages; p0 += kScan) {
        const int p = p0 + (int)threadIdx.x;
        (void)block_scan(p < pages && refs[p] > 0, lds, total);
        count += total;
    }
    int high = 0, hole = 0;
    for (int p0 = 0; p0 < pages; p0 += kScan) {
        const int p = p0 + (int)threadIdx.x;
        const int r = p < pages ? refs[p] : 0;
        const bool up = p < pages && r > 0 && p >= count, down = p < pages && r <= 0 && p < count;
        int ups, downs;
        const int a = high + block_scan(up, lds, ups), b = hole + block_scan(down, lds, downs);
        if (up) src[a] = p;
        if (down) dst[b] = p;
        if (p < pages) {
            if (!up) remap[p] = r > 0 ? p : -1;
            if (!down) refs_out[p] = p < count ? r : 0;
        }
        high += ups, hole += downs;
    }
    __threadfence_block();
    __syncthreads();
    for (int m = threadIdx.x; m < high; m += kScan) {
        remap[src[m]] = dst[m];
        refs_out[dst[m]] = refs[src[m]];
    }
    if (threadIdx.x == 0) *live = count, plan[0] = high;
}

template <typename V>
__global__ __launch_bounds__(256) void compact_kernel(uint8_t *cache, const int32_t *tables, int32_t *tables_out,
                                                      const int32_t *__restrict__ remap, const int32_t *__restrict__ plan,
                                                      int64_t entries, int layers, int64_t pages, int64_t page_bytes,
                                                      int64_t span) {
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (int64_t)gridDim.x * blockDim.x) {
        const int t = tables[e];
        tables_out[e] = t >= 0 && t < pages ? remap[t] : -1;
    }
    const int64_t count = plan[0];
    if (count) move_pages<V, true>(cache, plan + 4, plan + 4 + pages, count, layers, pages, page_bytes, span, blockIdx.x, gridDim.x);
}

int32_t sizes_ok(int layers, int64_t pages, int64_t page_bytes, int ps, int rows, int max_pages) {
    if (layers < 1 || pages < 1 || page_bytes < 1 || ps < 1 || rows < 1 || max_pages < 1) return kInvalid;
    if (pages > 0x3fffffff) return kUnsupported;
    return kOk;
}

constexpr int64_t kSpan = 16384;

// 16-byte units where pages and cache allow them
bool wide(const void *cache, int64_t page_bytes) { return ((uintptr_t)cache & 15u) == 0 && page_bytes % 16 == 0; }

// Up to 16 workgroups a CU, which take spans in turn.
unsigned copy_grid(int64_t moves, int layers, int64_t page_bytes) {
    const int64_t units = moves * layers * ((page_bytes + kSpan - 1) / kSpan);
    return (unsigned)(units < 1 ? 1 : units < 4096 ? units : 4096);
}

}  // namespace
}  // namespace bk

using namespace bk;

extern "C" int32_t baracuda_kernels_kv_pages_gfx950_can_implement(int32_t layers, int64_t num_pages, int64_t page_bytes,
                                                                  int32_t page_size, int32_t rows, int32_t max_pages) {
    return sizes_ok(layers, num_pages, page_bytes, page_size, rows, max_pages);
}

extern "C" size_t baracuda_kernels_kv_pages_gfx950_workspace_size(int32_t layers, int64_t num_pages, int64_t page_bytes,
                                                                  int32_t page_size, int32_t rows, int32_t max_pages) {
    if (sizes_ok(layers, num_pages, page_bytes, page_size, rows, max_pages) != kOk) return 0;
    return (size_t)(16 + 8 * num_pages);
}

extern "C" int32_t baracuda_kernels_kv_pages_copy_gfx950_run(int32_t layers, int64_t num_pages, int64_t page_bytes,
                                                             int64_t count, void *cache, const int32_t *src,
                                                             const int32_t *dst, void *stream) {
    const int32_t st = sizes_ok(layers, num_pages, page_bytes, 1, 1, 1);
    if (st != kOk) return st;
    if (count < 0) return kInvalid;
    if (count == 0) return kOk;
    if (!cache || !src || !dst) return kInvalid;
    const dim3 grid(copy_grid(count, layers, page_bytes));
    if (wide(cache, page_bytes))
        hipLaunchKernelGGL((copy_kernel<v4i>), grid, dim3(256), 0, (hipStream_t)stream, (uint8_t *)cache, src, dst, count,
                           layers, num_pages, page_bytes, kSpan);
    else
        hipLaunchKernelGGL((copy_kernel<uint8_t>), grid, dim3(256), 0, (hipStream_t)stream, (uint8_t *)cache, src, dst,
                           count, layers, num_pages, page_bytes, kSpan);
    return launch_status();
}

extern "C" int32_t baracuda_kernels_kv_pages_fork_gfx950_run(int32_t layers, int64_t num_pages, int64_t page_bytes,
                                                             int32_t page_size, int32_t rows, int32_t max_pages,
                                                             int32_t count, void *cache, int32_t *tables, int32_t *lens,
                                                             int32_t *refs, const int32_t *parents,
                                                             const int32_t *children, int32_t *fresh, void *stream) {
    const int32_t st = sizes_ok(layers, num_pages, page_bytes, page_size, rows, max_pages);
    if (st != kOk) return st;
    if (count < 0) return kInvalid;
    if (count > 65536) return kUnsupported;
    if (count == 0) return kOk;
    if (!cache || !tables || !lens || !refs || !parents || !children || !fresh) return kInvalid;
    const hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kScan), 0, s, lens, refs, parents, children, fresh, count, rows,
                       (int)num_pages, page_size, max_pages);
    const int32_t first = launch_status();
    if (first != kOk) return first;
    const dim3 grid((unsigned)count + copy_grid(count, layers, page_bytes));
    if (wide(cache, page_bytes))
        hipLaunchKernelGGL((fork_kernel<v4i>), grid, dim3(256), 0, s, (uint8_t *)cache, tables, lens, refs, parents,
                           children, fresh, count, rows, max_pages, page_size, layers, num_pages, page_bytes, kSpan);
    else
        hipLaunchKernelGGL((fork_kernel<uint8_t>), grid, dim3(256), 0, s, (uint8_t *)cache, tables, lens, refs, parents,
                           children, fresh, count, rows, max_pages, page_size, layers, num_pages, page_bytes, kSpan);
    return launch_status();
}

extern "C" int32_t baracuda_kernels_kv_pages_release_gfx950_run(int64_t num_pages, int32_t rows, int32_t max_pages,
                                                                int32_t count, int32_t *tables, int32_t *lens,
                                                                int32_t *refs, const int32_t *which, void *stream) {
    const int32_t st = sizes_ok(1, num_pages, 1, 1, rows, max_pages);
    if (st != kOk) return st;
    if (count < 0) return kInvalid;
    if (count > 0x7fffff) return kUnsupported;    // a launch has less than 2^32 threads
    if (count == 0) return kOk;
    if (!tables || !lens || !refs || !which) return kInvalid;
    const unsigned y = (unsigned)((max_pages + 255) / 256);
    hipLaunchKernelGGL(release_kernel, dim3((unsigned)count, y < 64 ? y : 64), dim3(256), 0, (hipStream_t)stream, tables,
                       lens, refs, which, rows, max_pages, (int)num_pages);
    return launch_status();
}

extern "C" int32_t baracuda_kernels_kv_pages_compact_gfx950_run(
    int32_t layers, int64_t num_pages, int64_t page_bytes, int32_t page_size, int32_t rows, int32_t max_pages, void *cache,
    const int32_t *tables, const int32_t *refs, int32_t *tables_out, int32_t *refs_out, int32_t *remap, int32_t *live,
    void *workspace, size_t workspace_bytes, void *stream) {
    const int32_t st = sizes_ok(layers, num_pages, page_bytes, page_size, rows, max_pages);
    if (st != kOk) return st;
    if (!cache || !tables || !refs || !tables_out || !refs_out || !remap || !live || refs == refs_out) return kInvalid;
    if (!workspace || workspace_bytes < (size_t)(16 + 8 * num_pages)) return kWorkspace;
    if ((uintptr_t)workspace & 3u) return kMisaligned;
    const hipStream_t s = (hipStream_t)stream;
    int32_t *plan = (int32_t *)workspace;
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kScan), 0, s, refs, refs_out, remap, live, plan, (int)num_pages);
    const int32_t first = launch_status();
    if (first != kOk) return first;
    const int64_t entries = (int64_t)rows * max_pages;
    // at most half the pages move
    const dim3 grid(copy_grid((num_pages + 1) / 2, layers, page_bytes));
    if (wide(cache, page_bytes))
        hipLaunchKernelGGL((compact_kernel<v4i>), grid, dim3(256), 0, s, (uint8_t *)cache, tables, tables_out, remap, plan,
                           entries, layers, num_pages, page_bytes, kSpan);
    else
        hipLaunchKernelGGL((compact_kernel<uint8_t>), grid, dim3(256), 0, s, (uint8_t *)cache, tables, tables_out, remap,
                           plan, entries, layers, num_pages, page_bytes, kSpan);
    return launch_status();
}
