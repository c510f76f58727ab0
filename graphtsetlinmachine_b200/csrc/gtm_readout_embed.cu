// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   forward:  out[b]  = scale * sum over the ids i of bag b of table[ids[i]]        (no bags: one id each)
//   gradient: dtab[r] = scale * sum over the positions i with ids[i] = r of grad[bag of i]
//
// Both are one operation: rows gathered by an index list that is cut into segments, each segment added up in 32 bits and
// rounded once.  Forward the list is `ids` and the segments are the bags; for the gradient the list is the bag of every
// position, sorted by id (stable radix sort), and the segments are the table's rows.  Sums have one order, that of the list, in
// pieces of kPiece: there are no atomics and results do not change from run to run.
#include "gtm_readout.cuh"

namespace gtm_readout {
namespace {

// A warp adds up to kPiece rows.  Longer segments leave their first kPiece rows in `head` and the rest in `part`, one slot
// per kPiece positions of the list: at most one such segment begins in a span of kPiece positions, and at most one goes on
// through it, so that a slot has one owner.
constexpr int kPiece = 128;

struct GatherArgs {
    const void *src;
    long long src_stride, rows;      // elements, rows of src
    const void *list;                // row of src per position
    int list_wide;
    const void *offsets;             // segments [offsets[s], offsets[s + 1]) of the list; null: one position each
    int offsets_wide;
    long long positions, segments;
    int columns;
    float scale;
    void *out;
    long long out_stride;
    float *head, *part;              // [spans][columns]
};

__device__ __forceinline__ long long clamp_offset(const GatherArgs &a, long long s)
{
    const long long o = index_at(a.offsets, a.offsets_wide, s);
    return o < 0 ? 0 : o > a.positions ? a.positions : o;
}

// Last segment that begins at or before `position`; -1: none does.
__device__ long long segment_at(const GatherArgs &a, long long position)
{
    long long low = -1, high = a.segments;        // offsets[low] <= position < offsets[high]
    while (high - low > 1) {
        const long long mid = (low + high) / 2;
        if (clamp_offset(a, mid) <= position) low = mid;
        else high = mid;
    }
    return low;
}

// Columns of a lane: U runs of V next to each other, 32 lanes of V apart.
template <class T, int V, int U>
__device__ __forceinline__ void add_rows(const GatherArgs &a, long long begin, long long end, int column0, float (&acc)[U][V])
{
    const int lane = threadIdx.x & 31;
    const T *src = (const T *)a.src;
    for (long long base = begin; base < end; base += 32) {
        const int n = (int)min(32ll, end - base);
        long long mine = -1;
        if (lane < n) mine = index_at(a.list, a.list_wide, base + lane);
        constexpr int kAhead = V * U * sizeof(T) >= 32 ? 4 : 8;
        for (int i = 0; i < n; i += kAhead) {
            Pack<T, V> got[kAhead][U];
            long long row[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                row[k] = __shfl_sync(~0u, mine, (i + k) & 31);
                if (i + k >= n) row[k] = -1;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int c = column0 + (u * 32 + lane) * V;
                    if (row[k] >= 0 && row[k] < a.rows && c < a.columns)
                        got[k][u] = *(const Pack<T, V> *)(src + row[k] * a.src_stride + c);
                    else
#pragma unroll
                        for (int v = 0; v < V; v++) got[k][u].v[v] = from_float<T>(0.f);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int v = 0; v < V; v++)
                        acc[u][v] += row[k] >= a.rows ? __int_as_float(0x7fffffff) : to_float(got[k][u].v[v]);
        }
    }
}

template <class T, int V, int U>
__global__ void __launch_bounds__(256) gather_sum_kernel(const GatherArgs a)
{
    const long long unit = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    const int lane = threadIdx.x & 31, column0 = blockIdx.y * (32 * V * U);
    const long long spans = a.offsets ? (a.positions + kPiece - 1) / kPiece : 0;
    long long begin, end;
    float *to = nullptr;
    if (unit < a.segments) {
        begin = a.offsets ? clamp_offset(a, unit) : unit;
        end = a.offsets ? clamp_offset(a, unit + 1) : unit + 1;
        if (end - begin > kPiece) {
            to = a.head + begin / kPiece * a.columns;
            end = begin + kPiece;
        }
    } else {
        if (a.positions <= kPiece || unit >= a.segments + spans) return;
        const long long span = unit - a.segments, s = segment_at(a, span * kPiece);
        if (s < 0) return;
        begin = max(span * kPiece, clamp_offset(a, s) + kPiece);
        end = min((span + 1) * kPiece, clamp_offset(a, s + 1));
        if (begin >= end) return;
        to = a.part + span * a.columns;
    }
    float acc[U][V];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < V; v++) acc[u][v] = 0.f;
    add_rows<T, V, U>(a, begin, end, column0, acc);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int c = column0 + (u * 32 + lane) * V;
        if (c >= a.columns) continue;
        if (to) {
#pragma unroll
            for (int v = 0; v < V; v++) to[c + v] = acc[u][v];
        } else {
            Pack<T, V> p;
#pragma unroll
            for (int v = 0; v < V; v++) p.v[v] = from_float<T>(acc[u][v] * a.scale);
            *(Pack<T, V> *)((T *)a.out + unit * a.out_stride + c) = p;
        }
    }
}

// Segments longer than kPiece: head and parts, added in the order of the list.  A block has the segment that begins in one span
// (if one does) and 32 columns; its eight warps take every eighth part and are added in order.
template <class T>
__global__ void __launch_bounds__(256) gather_join_kernel(const GatherArgs a)
{
    __shared__ float sums[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, c = blockIdx.y * 32 + lane;
    const long long span = blockIdx.x, last = min((span + 1) * kPiece, a.positions) - 1;
    const long long s = segment_at(a, last);
    if (s < 0) return;
    const long long begin = clamp_offset(a, s), end = clamp_offset(a, s + 1);
    if (begin < span * kPiece || end - begin <= kPiece) return;
    const long long first = (begin + kPiece) / kPiece, n = (end - 1) / kPiece - first + 1;
    float sum = 0.f;
    if (c < a.columns)
#pragma unroll 8
        for (long long i = warp; i < n; i += 8) sum += a.part[(first + i) * a.columns + c];
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || c >= a.columns) return;
    sum = a.head[span * a.columns + c];
#pragma unroll
    for (int w = 0; w < 8; w++) sum += sums[w][lane];
    ((T *)a.out)[s * a.out_stride + c] = from_float<T>(sum * a.scale);
}

template <class T, int V, int U>
int launch_gather(const GatherArgs &a, cudaStream_t stream)
{
    const bool long_ones = a.offsets && a.positions > kPiece;
    const long long spans = long_ones ? (a.positions + kPiece - 1) / kPiece : 0, units = a.segments + spans;
    const int wide = 32 * V * U;
    const dim3 grid((unsigned)((units + 7) / 8), (unsigned)((a.columns + wide - 1) / wide));
    gather_sum_kernel<T, V, U><<<grid, 256, 0, stream>>>(a);
    GTM_CU(cudaGetLastError());
    if (long_ones) {
        gather_join_kernel<T><<<dim3((unsigned)spans, (unsigned)((a.columns + 31) / 32)), 256, 0, stream>>>(a);
        GTM_CU(cudaGetLastError());
    }
    return GTM_OK;
}

// The widest loads that rows of both arrays start at a boundary of.
int launch_gather(const GatherArgs &a, int type, cudaStream_t stream)
{
    const int64_t size = (int64_t)type_bytes(type);
    const auto fits = [&](unsigned bytes) {
        return aligned(a.src, a.src_stride * size, bytes) && aligned(a.out, a.out_stride * size, bytes) && a.columns * size % bytes == 0;
    };
    if (type == GTM_F32) return fits(16) ? launch_gather<float, 4, 1>(a, stream) : launch_gather<float, 1, 4>(a, stream);
    if (type == GTM_BF16)
        return fits(16) ? launch_gather<__nv_bfloat16, 8, 1>(a, stream)
             : fits(4)  ? launch_gather<__nv_bfloat16, 2, 4>(a, stream) : launch_gather<__nv_bfloat16, 1, 8>(a, stream);
    return fits(16) ? launch_gather<__half, 8, 1>(a, stream)
         : fits(4)  ? launch_gather<__half, 2, 4>(a, stream) : launch_gather<__half, 1, 8>(a, stream);
}

// ------------------------------------------------------------------------------------ ids sorted, for the gradient
// Radix sort by digits of kDigit bits, the lowest first, of (id, bag) pairs; every pass keeps the order of equal digits.
// Ids that the table does not have (padding, too large ones, positions outside every bag) sort behind its last row.
constexpr int kDigit = 8, kDigits = 1 << kDigit, kSortThreads = 256, kPerThread = 16, kTile = kSortThreads * kPerThread;

__global__ void __launch_bounds__(256) sort_keys_kernel(const void *ids, int ids_wide, long long n, const void *offsets, int offsets_wide,
                                                        long long bags, unsigned rows, uint2 *pairs)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long id = index_at(ids, ids_wide, i);
    unsigned key = id < 0 || id >= (long long)rows ? rows : (unsigned)id, bag = (unsigned)i;
    if (offsets) {
        GatherArgs a;
        a.offsets = offsets, a.offsets_wide = offsets_wide, a.positions = n, a.segments = bags;
        const long long s = segment_at(a, i);
        if (s < 0 || i >= clamp_offset(a, s + 1)) key = rows;
        bag = s < 0 ? 0 : (unsigned)s;
    }
    pairs[i] = make_uint2(key, bag);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const uint2 *pairs, long long n, int shift, unsigned *counts)
{
    __shared__ unsigned hist[kDigits];
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) hist[d] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * kTile;
    for (int k = 0; k < kPerThread; k++) {
        const long long i = first + k * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&hist[(pairs[i].x >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) counts[(long long)d * gridDim.x + blockIdx.x] = hist[d];
}

// Exclusive running sums of all counts, digit by digit, block by block.  One block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(unsigned *counts, long long n)
{
    __shared__ unsigned warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const long long per = (n + 1023) / 1024, first = per * threadIdx.x, last = min(n, first + per);
    unsigned sum = 0;
    for (long long i = first; i < last; i++) sum += counts[i];
    unsigned run = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const unsigned v = __shfl_up_sync(~0u, run, o);
        if (lane >= o) run += v;
    }
    if (lane == 31) warp_sums[warp] = run;
    __syncthreads();
    if (warp == 0) {
        unsigned w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const unsigned v = __shfl_up_sync(~0u, w, o);
            if (lane >= o) w += v;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    run += (warp ? warp_sums[warp - 1] : 0u) - sum;
    for (long long i = first; i < last; i++) {
        const unsigned c = counts[i];
        counts[i] = run;
        run += c;
    }
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const uint2 *pairs, long long n, int shift, const unsigned *counts, uint2 *sorted)
{
    __shared__ unsigned warp_hist[kSortThreads / 32][kDigits];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    for (int d = threadIdx.x; d < kSortThreads / 32 * kDigits; d += kSortThreads) (&warp_hist[0][0])[d] = 0;
    __syncthreads();
    // a warp has kPerThread * 32 pairs in a row, 32 at a time: equal digits keep their order
    const long long first = (long long)blockIdx.x * kTile + warp * (kPerThread * 32) + lane;
    uint2 pair[kPerThread];
    unsigned rank[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; k++)
        if (first + k * 32 < n) pair[k] = pairs[first + k * 32];
#pragma unroll
    for (int k = 0; k < kPerThread; k++) {
        const bool real = first + k * 32 < n;
        const unsigned digit = real ? (pair[k].x >> shift) & (kDigits - 1) : kDigits;
        const unsigned peers = __match_any_sync(~0u, digit);
        const unsigned before = __popc(peers & ((1u << lane) - 1));
        if (real) rank[k] = warp_hist[warp][digit] + before;
        __syncwarp();
        if (real && before == 0) warp_hist[warp][digit] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
        unsigned run = counts[(long long)d * gridDim.x + blockIdx.x];
        for (int w = 0; w < kSortThreads / 32; w++) {
            const unsigned c = warp_hist[w][d];
            warp_hist[w][d] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPerThread; k++)
        if (first + k * 32 < n) sorted[warp_hist[warp][(pair[k].x >> shift) & (kDigits - 1)] + rank[k]] = pair[k];
}

// Where each row's positions begin in the sorted list (offsets[rows]: where ids that are no row begin), and the list of bags.
__global__ void __launch_bounds__(256) sort_rows_kernel(const uint2 *sorted, long long n, long long rows, int *offsets, int *bags)
{
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t <= rows) {
        long long low = 0, high = n;
        while (low < high) {
            const long long mid = (low + high) / 2;
            if (sorted[mid].x < t) low = mid + 1;
            else high = mid;
        }
        offsets[t] = (int)low;
    }
    if (t < n) bags[t] = (int)sorted[t].y;
}

struct GradientSpace {
    uint64_t pairs[2], counts, offsets, bags, head, part, total;
    long long tiles, spans;
};

GradientSpace gradient_space(long long ids, long long rows, long long columns)
{
    GradientSpace s;
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) { const uint64_t here = at; at += round_up(bytes, 256); return here; };
    s.tiles = (ids + kTile - 1) / kTile;
    s.spans = (ids + kPiece - 1) / kPiece;
    s.pairs[0] = take(ids * 8);
    s.pairs[1] = take(ids * 8);
    s.counts = take(s.tiles * kDigits * 4);
    s.offsets = take((rows + 1) * 4);
    s.bags = take(ids * 4);
    s.head = take(ids > kPiece ? s.spans * columns * 4 : 0);
    s.part = take(ids > kPiece ? s.spans * columns * 4 : 0);
    s.total = at;
    return s;
}

int check_sizes(const char *what, int type, int64_t rows, int64_t columns, int64_t ids, int64_t bags)
{
    if (!type_bytes(type)) return fail(GTM_ERR_ARG, "%s: element type %d is none of GTM_F32, GTM_BF16, GTM_F16", what, type);
    if (rows < 1 || rows >= kMostRows - 1) return fail(GTM_ERR_ARG, "%s: a table of %lld rows", what, (long long)rows);
    if (columns < 1 || columns > (1 << 20)) return fail(GTM_ERR_ARG, "%s: rows of %lld columns (1 to 2^20)", what, (long long)columns);
    if (ids < 0 || ids >= kMostRows || bags < 0 || bags >= kMostRows)
        return fail(GTM_ERR_ARG, "%s: %lld ids in %lld bags (at most 2^31 - 1)", what, (long long)ids, (long long)bags);
    return GTM_OK;
}

}  // namespace
}  // namespace gtm_readout

using namespace gtm_readout;

extern "C" int gtm_embed_workspace(int64_t ids, int64_t columns, int bags, uint64_t *bytes_out)
{
    if (!bytes_out) return fail(GTM_ERR_ARG, "gtm_embed_workspace: null output");
    GTM_TRY(check_sizes("gtm_embed_workspace", GTM_F32, 1, columns, ids, 0));
    const uint64_t slots = bags && ids > kPiece ? (uint64_t)((ids + kPiece - 1) / kPiece) : 0;
    *bytes_out = 2 * round_up(slots * columns * 4, 256);
    return GTM_OK;
}

extern "C" int gtm_embed(int device, void *cuda_stream, int type, const void *table, int64_t rows, int64_t columns, int64_t row_stride, const void *ids,
                         int ids_64, int64_t number_of_ids, const void *offsets, int offsets_64, int64_t number_of_bags, float scale, void *out,
                         int64_t out_stride, void *workspace, uint64_t workspace_bytes)
{
    GTM_TRY(check_sizes("gtm_embed", type, rows, columns, number_of_ids, number_of_bags));
    const int64_t segments = offsets ? number_of_bags : number_of_ids;
    if (segments == 0) return GTM_OK;
    if (!table || !out || (!ids && number_of_ids)) return fail(GTM_ERR_ARG, "gtm_embed: null array");
    if (row_stride < 0 || out_stride < columns) return fail(GTM_ERR_ARG, "gtm_embed: row stride %lld of the table, %lld of the result", (long long)row_stride, (long long)out_stride);
    uint64_t need = 0;
    GTM_TRY(gtm_embed_workspace(number_of_ids, columns, offsets != nullptr, &need));
    if (workspace_bytes < need || (need && ((uintptr_t)workspace % 16 || !workspace)))
        return fail(GTM_ERR_ARG, "gtm_embed: workspace of %llu bytes, %llu needed (16-byte aligned)", (unsigned long long)workspace_bytes, (unsigned long long)need);
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    GatherArgs a;
    a.src = table, a.src_stride = row_stride, a.rows = rows;
    a.list = ids, a.list_wide = ids_64, a.positions = number_of_ids;
    a.offsets = offsets, a.offsets_wide = offsets_64, a.segments = segments;
    a.columns = (int)columns, a.scale = scale, a.out = out, a.out_stride = out_stride;
    a.head = (float *)workspace, a.part = (float *)((char *)workspace + need / 2);
    return launch_gather(a, type, (cudaStream_t)cuda_stream);
}

extern "C" int gtm_embed_gradient_workspace(int64_t ids, int64_t rows, int64_t columns, uint64_t *bytes_out)
{
    if (!bytes_out) return fail(GTM_ERR_ARG, "gtm_embed_gradient_workspace: null output");
    GTM_TRY(check_sizes("gtm_embed_gradient_workspace", GTM_F32, rows, columns, ids, 0));
    *bytes_out = gradient_space(ids, rows, columns).total;
    return GTM_OK;
}

extern "C" int gtm_embed_gradient(int device, void *cuda_stream, int type, const void *gradient, int64_t columns, int64_t gradient_stride,
                                  const void *ids, int ids_64, int64_t number_of_ids, const void *offsets, int offsets_64, int64_t number_of_bags,
                                  float scale, void *table_gradient, int64_t rows, int64_t row_stride, void *workspace, uint64_t workspace_bytes)
{
    GTM_TRY(check_sizes("gtm_embed_gradient", type, rows, columns, number_of_ids, number_of_bags));
    if (!table_gradient || (number_of_ids && (!ids || !gradient))) return fail(GTM_ERR_ARG, "gtm_embed_gradient: null array");
    if (gradient_stride < 0 || row_stride < columns)
        return fail(GTM_ERR_ARG, "gtm_embed_gradient: row stride %lld of the gradient, %lld of the result", (long long)gradient_stride, (long long)row_stride);
    const GradientSpace space = gradient_space(number_of_ids, rows, columns);
    if (workspace_bytes < space.total || !workspace || (uintptr_t)workspace % 16)
        return fail(GTM_ERR_ARG, "gtm_embed_gradient: workspace of %llu bytes, %llu needed (16-byte aligned)", (unsigned long long)workspace_bytes, (unsigned long long)space.total);
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    char *w = (char *)workspace;
    uint2 *from = (uint2 *)(w + space.pairs[0]), *to = (uint2 *)(w + space.pairs[1]);
    unsigned *counts = (unsigned *)(w + space.counts);
    const long long n = number_of_ids;
    if (n) {
        sort_keys_kernel<<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(ids, ids_64, n, offsets, offsets_64, number_of_bags, (unsigned)rows, from);
        GTM_CU(cudaGetLastError());
        for (int shift = 0; shift < 32 && ((uint64_t)rows >> shift) != 0; shift += kDigit) {
            sort_count_kernel<<<(unsigned)space.tiles, kSortThreads, 0, stream>>>(from, n, shift, counts);
            GTM_CU(cudaGetLastError());
            sort_scan_kernel<<<1, 1024, 0, stream>>>(counts, space.tiles * kDigits);
            GTM_CU(cudaGetLastError());
            sort_place_kernel<<<(unsigned)space.tiles, kSortThreads, 0, stream>>>(from, n, shift, counts, to);
            GTM_CU(cudaGetLastError());
            std::swap(from, to);
        }
    }
    const long long threads = rows + 1 > n ? rows + 1 : n;
    sort_rows_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, stream>>>(from, n, rows, (int *)(w + space.offsets), (int *)(w + space.bags));
    GTM_CU(cudaGetLastError());
    GatherArgs a;
    a.src = gradient, a.src_stride = gradient_stride, a.rows = offsets ? number_of_bags : n;
    a.list = w + space.bags, a.list_wide = 0, a.positions = n;
    a.offsets = w + space.offsets, a.offsets_wide = 0, a.segments = rows;
    a.columns = (int)columns, a.scale = scale, a.out = table_gradient, a.out_stride = row_stride;
    a.head = (float *)(w + space.head), a.part = (float *)(w + space.part);
    return launch_gather(a, type, stream);
}
