// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   forward:  out[b]  = scale * sum over the ids i of bag b of table[ids[i]]        (no bags: one id each)
//   gradient: dtab[r] = scale * sum over the positions i with ids[i] = r of grad[bag of i]
//
// Both are one operation: rows gathered by an index list that is cut into segments, each segment added up in 32 bits and
// rounded once.  Forward the list is `ids` and the segments are the bags; for the gradient the list is the bag of every
// position, sorted by id (stable radix sort), and the segments are the table's rows.  Sums have one order, that of the list, in
// pieces of a span: there are no atomics on values and results do not change from run to run.
#include "gtm_readout.cuh"

#include <type_traits>
#include <utility>

namespace gtm_readout {
namespace {

// The list is cut into spans of 32, 64 or 128 positions, and a team of 4 to 32 lanes (as many as have a row's columns, 16 bytes each) adds up
// the rows of one span, whatever the segments are: teams have equal work with one id in a segment or a million.  A segment that
// goes on from one span to the next leaves its sums in 32 bits: the first in `head`, the others in `part`, one slot per
// span each, since only one segment can enter a span and one leave it.  `ends[span]` is the segment that entered it and ends there (-1:
// none); a second kernel adds its slots in order.  Segments without positions are zeroed by other teams.
struct GatherArgs {
    const void *src;
    long long src_stride, rows;      // elements, rows of src
    const uint2 *pairs;              // (segment, row of src) of every position, or null: from list and offsets
    const void *list;                // row of src per position
    int list_wide;
    const void *offsets;             // segments [offsets[s], offsets[s + 1]) of the list
    int offsets_wide;
    long long positions, segments;
    int columns, span;
    long long spans;
    float scale;
    void *out;
    long long out_stride;
    float *head, *part;              // [spans][partial_stride]
    int partial_stride;
    int *ends;
};

__device__ __forceinline__ long long clamp_offset(const void *offsets, int wide, long long positions, long long s)
{
    const long long o = index_at(offsets, wide, s);
    return o < 0 ? 0 : o > positions ? positions : o;
}

// Last segment that begins at or before `position`; -1: none does.  kLanes lanes ask together.
template <int kLanes>
__device__ long long segment_at(const void *offsets, int wide, long long positions, long long segments, long long position, unsigned team)
{
    const int lane = threadIdx.x % kLanes;
    long long low = -1, high = segments;          // offsets[low] <= position < offsets[high]
    while (high - low > 1) {
        const long long step = (high - low - 1 + kLanes - 1) / kLanes, at = low + 1 + lane * step;
        const unsigned before = __ballot_sync(team, at < high && clamp_offset(offsets, wide, positions, at) <= position);
        const int n = __popc(before & team);      // offsets do not decrease: the first n lanes
        if (n < kLanes) high = min(high, low + 1 + n * step);
        if (n > 0) low = low + 1 + (n - 1) * step;
    }
    return low;
}

// Segment of a position at or behind the beginning of segment `from` (-1: of none), -1 where it is in none.  Mostly the same or one
// of the next; behind many empty ones, found by halves.
__device__ __forceinline__ long long segment_from(const void *offsets, int wide, long long positions, long long segments, long long &from, long long position)
{
    for (int tries = 0; tries < 8 && from + 1 < segments && clamp_offset(offsets, wide, positions, from + 1) <= position; tries++) from++;
    long long high = segments;
    if (from + 1 < segments && clamp_offset(offsets, wide, positions, from + 1) <= position)
        while (high - from > 1) {
            const long long mid = (from + high) / 2;
            if (clamp_offset(offsets, wide, positions, mid) <= position) from = mid;
            else high = mid;
        }
    return from >= 0 && position < clamp_offset(offsets, wide, positions, from + 1) ? from : -1;
}

__device__ __forceinline__ void add2(float2 &a, float x, float y)
{
    unsigned long long &s = reinterpret_cast<unsigned long long &>(a);
    const float2 b = make_float2(x, y);
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s) : "l"(reinterpret_cast<const unsigned long long &>(b)));
}

// Values of a pack as floats, two at a time.
template <class T, int V>
__device__ __forceinline__ void accumulate(float2 (&acc)[(V + 1) / 2], const Pack<T, V> &p)
{
    if constexpr (V == 1) acc[0].x += to_float(p.v[0]);
    else
#pragma unroll
        for (int v = 0; v < V; v += 2) add2(acc[v / 2], to_float(p.v[v]), to_float(p.v[v + 1]));
}

// Four rows ahead at 28 warps an SM, eight at 20: 72 us and 80 for 819,200 rows of 256 bf16 in bags of 200.  kLong: 64 us (6.6 TB/s, from L2)
// and 45 for the gradient of 65,539 rows of 512 fp16 in segments of two; otherwise 72 and 33.  At 28 warps a thread has 72 registers, which the bf16 variants of 16-byte loads do
// not get by with (kLong: up to 400 bytes spilled; fp16 24, fp32 4): fp16 takes 49 us (8.5 TB/s) for what bf16 takes 64.
constexpr int kGatherThreads = 128, kGatherBlocks = 7;

// A lane has U runs of V columns next to each other, kLanes * V apart.  kLong: segments of several rows, taken one after the other; otherwise rows
// are loaded whatever their segments are, and each is asked for its own.  The order of the sums is the same.
template <class T, int V, int U, int kLanes, bool kLong>
__global__ void __launch_bounds__(kGatherThreads, U == 1 ? kGatherBlocks : 3) gather_sum_kernel(const GatherArgs a)
{
    next_may_start();
    wait_for_previous();
    constexpr int kColumns = kLanes * V * U, kAhead = 4;
    const int lane = threadIdx.x % kLanes, column0 = blockIdx.y * kColumns;
    const unsigned team = kLanes == 32 ? ~0u : ((1u << kLanes % 32) - 1) << ((threadIdx.x & 31) / kLanes * kLanes);
    const long long unit = (long long)blockIdx.x * (kGatherThreads / kLanes) + threadIdx.x / kLanes;
    float2 acc[U][(V + 1) / 2];
    bool bad = false;                             // an id beyond the table
    const auto clear = [&] {
        bad = false;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int v = 0; v < (V + 1) / 2; v++) acc[u][v] = make_float2(0.f, 0.f);
    };
    const auto write = [&](long long segment) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = column0 + (u * kLanes + lane) * V;
            if (c >= a.columns) continue;
            Pack<T, V> p;
#pragma unroll
            for (int v = 0; v < V; v++) p.v[v] = from_float<T>(bad ? __int_as_float(0x7fffffff) : (v % 2 ? acc[u][v / 2].y : acc[u][v / 2].x) * a.scale);
            *(Pack<T, V> *)((T *)a.out + segment * a.out_stride + c) = p;
        }
    };
    clear();
    if (unit >= a.spans) {
        // zeros of kLanes segments
        const long long first = (unit - a.spans) * kLanes, mine = first + lane;
        const bool none = mine < a.segments && clamp_offset(a.offsets, a.offsets_wide, a.positions, mine) >= clamp_offset(a.offsets, a.offsets_wide, a.positions, mine + 1);
        for (unsigned which = (__ballot_sync(team, none) & team) >> ((threadIdx.x & 31) / kLanes * kLanes); which; which &= which - 1) write(first + __ffs(which) - 1);
        return;
    }
    const T *column[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int c = column0 + (u * kLanes + lane) * V;
        column[u] = (const T *)a.src + (c < a.columns ? c : 0);      // lanes behind the last column read the first one, and drop it
    }
    const long long first = unit * a.span, last = min(first + a.span, a.positions);
    long long base = -1;                          // a segment at or before the lane's next position
    if (!a.pairs) base = segment_at<kLanes>(a.offsets, a.offsets_wide, a.positions, a.segments, first ? first - 1 : 0, team);
    const auto segment_of = [&](long long position) -> int {
        if (a.pairs) return a.pairs[position].x < (unsigned long long)a.segments ? (int)a.pairs[position].x : -1;
        return (int)segment_from(a.offsets, a.offsets_wide, a.positions, a.segments, base, position);
    };
    int now = first ? segment_of(first - 1) : -1, entered = now, ended = -1;      // a segment that is -1 is none
    const auto leave = [&](bool goes_on) {
        if (now >= 0) {
            if (now != entered && !goes_on) write(now);
            else {
                float *to = (now == entered ? a.part : a.head) + unit * a.partial_stride;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const int c = column0 + (u * kLanes + lane) * V + v;
                        if (c < a.columns) to[c] = bad ? __int_as_float(0x7fffffff) : v % 2 ? acc[u][v / 2].y : acc[u][v / 2].x;
                    }
                if (now == entered && !goes_on) ended = now;
            }
        }
        clear();
    };
    bool begun = false;                           // whether the span has a position of `now`
    int next_row = -1, next_segment = -1;         // of the lane's next position, read before the rows of the positions at hand
    const auto look = [&](long long position) {
        next_row = next_segment = -1;
        if (position >= last) return;
        if (a.pairs) {
            const uint2 pair = a.pairs[position];
            next_segment = pair.x < (unsigned long long)a.segments ? (int)pair.x : -1, next_row = (int)pair.y;
        } else {
            const long long id = index_at(a.list, a.list_wide, position);
            next_segment = segment_of(position);
            next_row = id >= a.rows ? -2 : id < 0 ? -1 : (int)id;
        }
        if (next_segment < 0) next_row = -1;
    };
    look(first + lane);
    for (long long at = first; at < last; at += kLanes) {
        const int row = next_row, segment = next_segment;
        look(at + kLanes + lane);
        const int n = (int)min((long long)kLanes, last - at);
        const auto enter = [&](int next) {
            if (next == now) return;
            if (begun) leave(false);
            else entered = -1;                                    // it ended with the span before
            now = next;
        };
        enter(__shfl_sync(team, segment, 0, kLanes));
        begun = true;
        if constexpr (kLong) {
            // one segment after the other, kAhead rows at once
            const int shift = (threadIdx.x & 31) / kLanes * kLanes, before = __shfl_up_sync(team, segment, 1, kLanes);
            const unsigned changes = (__ballot_sync(team, lane > 0 && lane < n && segment != before) & team) >> shift;
            const bool whole = __all_sync(team, row >= 0 || lane >= n);
            for (int i = 0; i < n;) {
                const unsigned later = changes & ~((2u << i) - 1);
                const int j = later ? __ffs(later) - 1 : n;
                enter(__shfl_sync(team, segment, i, kLanes));
#pragma unroll 1
                for (; whole && i + kAhead <= j; i += kAhead) {
                    Pack<T, V> got[kAhead][U];
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        const unsigned long long from = (unsigned long long)(unsigned)__shfl_sync(team, row, i + k, kLanes) * (unsigned)a.src_stride;
#pragma unroll
                        for (int u = 0; u < U; u++) got[k][u] = *(const Pack<T, V> *)(column[u] + from);
                    }
#pragma unroll
                    for (int k = 0; k < kAhead; k++)
#pragma unroll
                        for (int u = 0; u < U; u++) accumulate<T, V>(acc[u], got[k][u]);
                }
#pragma unroll 1
                for (; i < j; i += kAhead) {
                    Pack<T, V> got[kAhead][U];
                    int which[kAhead];
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        which[k] = __shfl_sync(team, row, i + k, kLanes);
                        if (i + k >= j) which[k] = -1;
                        if (which[k] >= 0)
#pragma unroll
                            for (int u = 0; u < U; u++) got[k][u] = *(const Pack<T, V> *)(column[u] + (unsigned long long)(unsigned)which[k] * (unsigned)a.src_stride);
                    }
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        if (which[k] >= 0)
#pragma unroll
                            for (int u = 0; u < U; u++) accumulate<T, V>(acc[u], got[k][u]);
                        bad |= which[k] == -2;
                    }
                }
                i = j;
            }
        } else {
            if (n == kLanes && __all_sync(team, segment == now && row >= 0)) {
                // all of one segment
#pragma unroll 1
                for (int i = 0; i < kLanes; i += kAhead) {
                    Pack<T, V> got[kAhead][U];
#pragma unroll
                    for (int k = 0; k < kAhead; k++) {
                        const unsigned long long from = (unsigned long long)(unsigned)__shfl_sync(team, row, i + k, kLanes) * (unsigned)a.src_stride;
#pragma unroll
                        for (int u = 0; u < U; u++) got[k][u] = *(const Pack<T, V> *)(column[u] + from);
                    }
#pragma unroll
                    for (int k = 0; k < kAhead; k++)
#pragma unroll
                        for (int u = 0; u < U; u++) accumulate<T, V>(acc[u], got[k][u]);
                }
                continue;
            }
#pragma unroll 1
            for (int i = 0; i < n; i += kAhead) {
                Pack<T, V> got[kAhead][U];
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    // a position without a row reads the first one, and drops it
                    const unsigned long long from = (unsigned long long)(unsigned)max(__shfl_sync(team, row, i + k, kLanes), 0) * (unsigned)a.src_stride;
                    if (a.rows > 0)
#pragma unroll
                        for (int u = 0; u < U; u++) got[k][u] = *(const Pack<T, V> *)(column[u] + from);
                }
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    const int next = __shfl_sync(team, segment, i + k, kLanes), which = __shfl_sync(team, row, i + k, kLanes);
                    if (i + k >= n) continue;
                    enter(next);
                    if (which >= 0)
#pragma unroll
                        for (int u = 0; u < U; u++) accumulate<T, V>(acc[u], got[k][u]);
                    else bad |= which == -2;
                }
            }
        }
    }
    // every lane's `base` is at or before its last position: any of them finds the next one's segment
    leave(last < a.positions && now >= 0 && segment_of(last) == now);
    if (blockIdx.y == 0 && lane == 0 && a.spans > 1) a.ends[unit] = ended;
}

// Segments of several spans: head and parts, added in the order of the list (7 us for 65,539 positions, bound by the way from one load to the next).  A warp has the segment that ends in its span (if one
// does) and 128 columns; where a segment has more than kAlone parts, the block's warps take them in turn.
template <class T>
__global__ void __launch_bounds__(256) gather_join_kernel(const GatherArgs a)
{
    next_may_start();
    wait_for_previous();
    constexpr int kAlone = 16, kWarps = 8;
    __shared__ float4 sums[kWarps][32];
    __shared__ long long longest[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, c = blockIdx.y * 128 + lane * 4;
    const long long span = (long long)blockIdx.x * kWarps + warp;
    const bool inside = c < a.partial_stride;
    const auto begin_of = [&](long long s) { return clamp_offset(a.offsets, a.offsets_wide, a.positions, s) / a.span; };
    const auto sum_of = [&](long long first, long long n, int step) {
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside)
#pragma unroll 8
            for (long long i = 0; i < n; i += step) {
                const float4 v = *(const float4 *)(a.part + (first + i) * a.partial_stride + c);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
        return sum;
    };
    const auto head_of = [&](long long unit) { return inside ? *(const float4 *)(a.head + unit * a.partial_stride + c) : make_float4(0.f, 0.f, 0.f, 0.f); };
    const auto write = [&](long long s, float4 head, float4 sum) {
        const float v[4] = {head.x + sum.x, head.y + sum.y, head.z + sum.z, head.w + sum.w};
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < a.columns) ((T *)a.out)[s * a.out_stride + c + k] = from_float<T>(v[k] * a.scale);
    };
    const long long s = span < a.spans ? a.ends[span] : -1;
    long long first = 0, n = 0;
    if (s >= 0) {
        first = begin_of(s) + 1;
        n = span - first + 1;
    }
    if (n > 0 && n <= kAlone) {
        const float4 head = head_of(first - 1);
        write(s, head, sum_of(first, n, 1));
    }
    if (lane == 0) longest[warp] = n > kAlone ? s : -1;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) {
        const long long one = longest[w];
        if (one < 0) continue;                  // the block together
        const long long begin = begin_of(one) + 1, parts = (long long)blockIdx.x * kWarps + w - begin + 1;
        sums[warp][lane] = sum_of(begin + warp, parts - warp, kWarps);
        __syncthreads();
        if (warp == 0) {
            float4 sum = sums[0][lane];
            for (int k = 1; k < kWarps; k++) sum.x += sums[k][lane].x, sum.y += sums[k][lane].y, sum.z += sums[k][lane].z, sum.w += sums[k][lane].w;
            write(one, head_of(begin - 1), sum);
        }
        __syncthreads();
    }
}

// Lanes that have a row's columns, 16 bytes each: as few as there are, so that a warp has several narrow rows.
int team_lanes(int64_t columns, size_t element)
{
    const int64_t wide = 16 / element;
    return columns <= 4 * wide ? 4 : columns <= 8 * wide ? 8 : columns <= 16 * wide ? 16 : 32;
}

// Long spans (fewer slots of sums) as long as there are 16 warps per SM of them.
int span_of(int64_t positions, int64_t columns, size_t element)
{
    if (positions <= 128) return 128;                 // one span: nothing to join
    const int lanes = team_lanes(columns, element);
    const int64_t blocks = (columns * element + lanes * 16 - 1) / (lanes * 16), teams = (int64_t)148 * 16 * 32 / lanes;
    for (int span = 128; span > 32; span /= 2)
        if (positions / span * blocks >= teams) return span;
    return 32;
}

int64_t partial_stride(int64_t columns) { return (int64_t)round_up(columns, 4); }

// Slots of sums, and where the segments end.
struct GatherSpace {
    uint64_t head, part, ends, total;
};

GatherSpace gather_space(uint64_t at, int64_t positions, int64_t columns)
{
    // of the shortest spans: a caller's workspace serves every element type.  What is one span needs none
    const uint64_t spans = positions <= 128 ? 0 : (uint64_t)(positions + 31) / 32, sums = round_up(spans * partial_stride(columns) * 4, 256);
    return {at, at + sums, at + 2 * sums, at + 2 * sums + round_up(spans * 4, 256)};
}

template <class T, int V, int U, int kLanes>
int launch_gather(const GatherArgs &a, cudaStream_t stream)
{
    constexpr int kLongRows = 8;         // rows of a segment, on the average
    constexpr int kWide = kLanes * V * U, kTeams = kGatherThreads / kLanes;
    const long long units = a.spans + (a.segments + kLanes - 1) / kLanes;
    const dim3 grid((unsigned)((units + kTeams - 1) / kTeams), (unsigned)((a.columns + kWide - 1) / kWide));
    const bool long_ones = a.positions >= a.segments * kLongRows;
    GTM_TRY(launch_early(long_ones ? gather_sum_kernel<T, V, U, kLanes, true> : gather_sum_kernel<T, V, U, kLanes, false>, grid, dim3(kGatherThreads), 0, stream, a));
    if (a.spans > 1) GTM_TRY(launch_early(gather_join_kernel<T>, dim3((unsigned)((a.spans + 7) / 8), (unsigned)((a.columns + 127) / 128)), dim3(256), 0, stream, a));
    return GTM_OK;
}

template <class T, int V>
int launch_lanes(const GatherArgs &a, cudaStream_t stream)
{
    constexpr int U = 16 / sizeof(T) / V;
    switch (team_lanes(a.columns, sizeof(T))) {
    case 4: return launch_gather<T, V, U, 4>(a, stream);
    case 8: return launch_gather<T, V, U, 8>(a, stream);
    case 16: return launch_gather<T, V, U, 16>(a, stream);
    default: return launch_gather<T, V, U, 32>(a, stream);
    }
}

// The widest loads that rows of both arrays start at a boundary of.  Which lane has a column changes with that, the order of a sum does not.
template <class T>
int launch_gather(const GatherArgs &a, cudaStream_t stream)
{
    const auto fits = [&](unsigned bytes) {
        return aligned(a.src, a.src_stride * sizeof(T), bytes) && aligned(a.out, a.out_stride * sizeof(T), bytes) && a.columns * sizeof(T) % bytes == 0;
    };
    if (fits(16)) return launch_lanes<T, 16 / sizeof(T)>(a, stream);
    if (sizeof(T) == 2 && fits(4)) return launch_lanes<T, 4 / sizeof(T)>(a, stream);
    return launch_lanes<T, 1>(a, stream);
}

int launch_gather(GatherArgs &a, int type, char *workspace, const GatherSpace &space, cudaStream_t stream)
{
    a.span = span_of(a.positions, a.columns, type_bytes(type));
    a.spans = (a.positions + a.span - 1) / a.span;
    a.head = (float *)(workspace + space.head), a.part = (float *)(workspace + space.part), a.ends = (int *)(workspace + space.ends);
    a.partial_stride = (int)partial_stride(a.columns);
    return type == GTM_F32 ? launch_gather<float>(a, stream) : type == GTM_BF16 ? launch_gather<__nv_bfloat16>(a, stream) : launch_gather<__half>(a, stream);
}

// Rows by id, without bags.  A thread makes 16 bytes of the result at a time, kEach of them at once: one load where the rows lie at
// 16-byte boundaries, single elements (of two rows, or of several short ones) where they do not, which the load units' rate then bounds: 22 us for 24,001
// rows of 1,001 bf16 (4.3 TB/s).  kNarrow: the result has fewer than 2^32 elements, and rows are found by a 32-bit division.
template <class T, bool kWhole, bool kNarrow>
__global__ void __launch_bounds__(256) embed_rows_kernel(const T *table, long long stride, long long rows, const void *ids, int ids_wide, long long count, int columns, float scale, T *out)
{
    next_may_start();
    wait_for_previous();
    constexpr int V = 16 / sizeof(T), kEach = kWhole ? 4 : 2;
    const long long all = count * columns, step = (long long)gridDim.x * 256 * V;
    for (long long first = ((long long)blockIdx.x * 256 + threadIdx.x) * V; first < all; first += step * kEach) {
        Pack<T, V> p[kEach];
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const long long at = first + e * step;
            if (at >= all) continue;
            long long row = kNarrow ? (long long)((unsigned)at / (unsigned)columns) : at / columns;
            int c = (int)(at - row * columns);
            long long id = index_at(ids, ids_wide, row);
            if constexpr (kWhole) {
                if (id >= 0 && id < rows) p[e] = *(const Pack<T, V> *)(table + id * stride + c);
                else
#pragma unroll
                    for (int v = 0; v < V; v++) p[e].v[v] = from_float<T>(id < 0 ? 0.f : __int_as_float(0x7fffffff));
            } else if (c + V <= columns) {
                // all of one row
                const bool real = id >= 0 && id < rows;
                const T *from = table + (real ? id : 0) * stride + c;
#pragma unroll
                for (int v = 0; v < V; v++) p[e].v[v] = from[v];
                if (!real)
#pragma unroll
                    for (int v = 0; v < V; v++) p[e].v[v] = from_float<T>(id < 0 ? 0.f : __int_as_float(0x7fffffff));
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    p[e].v[v] = from_float<T>(id < 0 ? 0.f : __int_as_float(0x7fffffff));
                    if (at + v < all) {
                        if (id >= 0 && id < rows) p[e].v[v] = table[id * stride + c];
                        if (++c == columns && at + v + 1 < all) c = 0, id = index_at(ids, ids_wide, ++row);
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const long long at = first + e * step;
            if (at >= all) continue;
#pragma unroll
            for (int v = 0; v < V; v++) p[e].v[v] = from_float<T>(to_float(p[e].v[v]) * scale);
            if (at + V <= all) *(Pack<T, V> *)(out + at) = p[e];
            else
#pragma unroll
                for (int v = 0; v < V; v++)
                    if (at + v < all) out[at + v] = p[e].v[v];
        }
    }
}

template <class T>
int launch_rows(const void *table, int64_t stride, int64_t rows, const void *ids, int ids_wide, int64_t count, int64_t columns, float scale, void *out, cudaStream_t stream)
{
    constexpr int64_t V = 16 / sizeof(T);
    const bool whole = aligned(table, stride * sizeof(T), 16) && columns % V == 0, narrow = count * columns < (int64_t)1 << 32;
    const int64_t chunks = (count * columns + V - 1) / V, blocks = (chunks + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);
    const auto kernel = whole ? (narrow ? embed_rows_kernel<T, true, true> : embed_rows_kernel<T, true, false>) : narrow ? embed_rows_kernel<T, false, true> : embed_rows_kernel<T, false, false>;
    return launch_early(kernel, dim3(grid), dim3(256), 0, stream, (const T *)table, (long long)stride, (long long)rows, ids, ids_wide, (long long)count, (int)columns, scale, (T *)out);
}

// ------------------------------------------------------------------------------------ ids sorted, for the gradient
// Radix sort by digits of kDigit bits, the lowest first, of (id, bag) pairs; every pass keeps the order of equal digits.
// Ids that the table does not have (padding, too large ones, positions outside every bag) sort behind its last row.  Counts, running
// sums and placing are kernels of their own; what bounds them is their number, 20 us for 65,539 ids and 55 for 819,200 in two digits.
// Every kernel of the chain may be set up while the one before it ends.
constexpr int kDigit = 8, kDigits = 1 << kDigit, kSortThreads = 256, kSortWarps = kSortThreads / 32;

// A warp has kEach * 32 pairs in a row, 32 at a time.
template <int kEach> __device__ __forceinline__ long long sort_first() { return (long long)blockIdx.x * (kSortThreads * kEach) + threadIdx.x / 32 * (kEach * 32) + (threadIdx.x & 31); }

__device__ __forceinline__ void sort_count(unsigned *hist, unsigned *counts)
{
    __syncthreads();
    counts[(long long)blockIdx.x * kDigits + threadIdx.x] = hist[threadIdx.x];
}

template <int kEach>
__global__ void __launch_bounds__(kSortThreads) sort_keys_kernel(const void *ids, int ids_wide, long long n, const void *offsets, int offsets_wide, long long bags, unsigned rows,
                                                                uint2 *pairs, unsigned *counts)
{
    next_may_start();
    wait_for_previous();
    __shared__ unsigned hist[kDigits];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const long long first = sort_first<kEach>(), lane = threadIdx.x & 31;
    long long base = -1;
    if (offsets && first - lane < n) base = segment_at<32>(offsets, offsets_wide, n, bags, first - lane, ~0u);
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const long long i = first + k * 32;
        if (i >= n) break;
        const long long id = index_at(ids, ids_wide, i), bag = offsets ? segment_from(offsets, offsets_wide, n, bags, base, i) : i;
        const unsigned key = bag < 0 || id < 0 || id >= (long long)rows ? rows : (unsigned)id;
        pairs[i] = make_uint2(key, bag < 0 ? 0 : (unsigned)bag);
        atomicAdd(&hist[key & (kDigits - 1)], 1u);
    }
    sort_count(hist, counts);
}

template <int kEach>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const uint2 *pairs, long long n, int shift, unsigned *counts)
{
    next_may_start();
    wait_for_previous();
    __shared__ unsigned hist[kDigits];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const long long first = sort_first<kEach>();
    unsigned key[kEach];
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (first + k * 32 < n) key[k] = pairs[first + k * 32].x;
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (first + k * 32 < n) atomicAdd(&hist[(key[k] >> shift) & (kDigits - 1)], 1u);
    sort_count(hist, counts);
}

// Counts [block][digit] become where each block's pairs of a digit go: running sums digit by digit, block by block.  One block;
// a thread has a digit and every fourth part of the blocks.
__global__ void __launch_bounds__(1024) sort_scan_kernel(unsigned *counts, int blocks)
{
    next_may_start();
    wait_for_previous();
    __shared__ unsigned sums[4][kDigits], warp_sums[8];
    const int digit = threadIdx.x & (kDigits - 1), part = threadIdx.x / kDigits, lane = threadIdx.x & 31;
    const int per = (blocks + 3) / 4, first = min(blocks, part * per), last = min(blocks, first + per);
    unsigned sum = 0;
#pragma unroll 8
    for (int b = first; b < last; b++) sum += counts[(long long)b * kDigits + digit];
    sums[part][digit] = sum;
    __syncthreads();
    unsigned all = 0, run = 0;
    if (part == 0) {
        all = sums[0][digit] + sums[1][digit] + sums[2][digit] + sums[3][digit];
        run = all;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const unsigned v = __shfl_up_sync(~0u, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) warp_sums[digit / 32] = run;
    }
    __syncthreads();
    if (part == 0) {
        for (int w = 0; w < digit / 32; w++) run += warp_sums[w];
        run -= all;
        for (int q = 0; q < 4; q++) {
            const unsigned c = sums[q][digit];
            sums[q][digit] = run;
            run += c;
        }
    }
    __syncthreads();
    run = sums[part][digit];
#pragma unroll 8
    for (int b = first; b < last; b++) {
        const unsigned c = counts[(long long)b * kDigits + digit];
        counts[(long long)b * kDigits + digit] = run;
        run += c;
    }
}

template <int kEach>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const uint2 *pairs, long long n, int shift, const unsigned *counts, uint2 *sorted)
{
    next_may_start();
    wait_for_previous();
    __shared__ unsigned warp_hist[kSortWarps][kDigits];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) warp_hist[w][threadIdx.x] = 0;
    const long long first = sort_first<kEach>();
    uint2 pair[kEach];
    unsigned rank[kEach];
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (first + k * 32 < n) pair[k] = pairs[first + k * 32];
    unsigned run = counts[(long long)blockIdx.x * kDigits + threadIdx.x];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; k++) {
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
#pragma unroll
    for (int w = 0; w < kSortWarps; w++) {
        const unsigned c = warp_hist[w][threadIdx.x];
        warp_hist[w][threadIdx.x] = run;
        run += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; k++)
        if (first + k * 32 < n) sorted[warp_hist[warp][(pair[k].x >> shift) & (kDigits - 1)] + rank[k]] = pair[k];
}

// Where each row's positions begin in the sorted list (offsets[rows]: where ids that are no row begin).  The
// pair at a position writes the offsets of the rows behind the pair before it; of many such rows, its warp does.
__global__ void __launch_bounds__(256) sort_rows_kernel(const uint2 *sorted, long long n, long long rows, int *offsets)
{
    next_may_start();
    wait_for_previous();
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const int lane = threadIdx.x & 31;
    long long low = 0, high = 0;                   // offsets [low, high) are t
    if (t <= n) {
        low = t == 0 ? 0 : (long long)sorted[t - 1].x + 1;
        high = t == n ? rows + 1 : (long long)sorted[t].x + 1;
    }
    if (high - low <= 8) {
        for (long long r = low; r < high; r++) offsets[r] = (int)t;
        high = low;
    }
    for (unsigned many = __ballot_sync(~0u, high > low); many; many &= many - 1) {
        const int from = __ffs(many) - 1;
        const long long first = __shfl_sync(~0u, low, from), last = __shfl_sync(~0u, high, from);
        const int value = (int)__shfl_sync(~0u, t, from);
        for (long long r = first + lane; r < last; r += 32) offsets[r] = value;
    }
}

struct GradientSpace {
    uint64_t pairs[2], counts, offsets, total;
    GatherSpace gather;
    long long tiles;
    int each;
};

GradientSpace gradient_space(long long ids, long long rows, long long columns)
{
    GradientSpace s;
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) { const uint64_t here = at; at += round_up(bytes, 256); return here; };
    // small blocks of pairs as long as they do not fill the GPU, large ones (fewer counts) then
    s.each = ids > 148 * 4 * kSortThreads * 4 ? 16 : 4;
    s.tiles = (ids + kSortThreads * s.each - 1) / (kSortThreads * s.each);
    s.pairs[0] = take(ids * 8);
    s.pairs[1] = take(ids * 8);
    s.counts = take(s.tiles * kDigits * 4);
    s.offsets = take((rows + 1) * 4);
    s.gather = gather_space(at, ids, columns);
    s.total = s.gather.total;
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
    *bytes_out = bags ? gather_space(0, ids, columns).total : 0;
    return GTM_OK;
}

extern "C" int gtm_embed(int device, void *cuda_stream, int type, const void *table, int64_t rows, int64_t columns, int64_t row_stride, const void *ids,
                         int ids_64, int64_t number_of_ids, const void *offsets, int offsets_64, int64_t number_of_bags, float scale, void *out,
                         void *workspace, uint64_t workspace_bytes)
{
    GTM_TRY(check_sizes("gtm_embed", type, rows, columns, number_of_ids, number_of_bags));
    const int64_t segments = offsets ? number_of_bags : number_of_ids;
    if (segments == 0) return GTM_OK;
    if (!table || !out || (!ids && number_of_ids)) return fail(GTM_ERR_ARG, "gtm_embed: null array");
    if ((uintptr_t)table % type_bytes(type) || (uintptr_t)ids % (ids_64 ? 8 : 4) || (uintptr_t)offsets % (offsets_64 ? 8 : 4))
        return fail(GTM_ERR_ARG, "gtm_embed: an array does not start at a boundary of its elements");
    if (row_stride < 0 || row_stride >= kMostRows) return fail(GTM_ERR_ARG, "gtm_embed: row stride %lld of the table", (long long)row_stride);
    if ((uintptr_t)out % 16) return fail(GTM_ERR_ARG, "gtm_embed: the result does not start at a 16-byte boundary");
    uint64_t need = 0;
    GTM_TRY(gtm_embed_workspace(number_of_ids, columns, offsets != nullptr, &need));
    if (workspace_bytes < need || (need && ((uintptr_t)workspace % 16 || !workspace)))
        return fail(GTM_ERR_ARG, "gtm_embed: workspace of %llu bytes, %llu needed (16-byte aligned)", (unsigned long long)workspace_bytes, (unsigned long long)need);
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    if (!offsets)
        return type == GTM_F32    ? launch_rows<float>(table, row_stride, rows, ids, ids_64, number_of_ids, columns, scale, out, stream)
               : type == GTM_BF16 ? launch_rows<__nv_bfloat16>(table, row_stride, rows, ids, ids_64, number_of_ids, columns, scale, out, stream)
                                  : launch_rows<__half>(table, row_stride, rows, ids, ids_64, number_of_ids, columns, scale, out, stream);
    GatherArgs a;
    a.src = table, a.src_stride = row_stride, a.rows = rows;
    a.list = ids, a.list_wide = ids_64, a.positions = number_of_ids;
    a.offsets = offsets, a.offsets_wide = offsets_64, a.segments = segments;
    a.columns = (int)columns, a.scale = scale, a.out = out, a.out_stride = columns;
    a.pairs = nullptr;
    return launch_gather(a, type, (char *)workspace, gather_space(0, number_of_ids, columns), stream);
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
                                  float scale, void *table_gradient, int64_t rows, void *workspace, uint64_t workspace_bytes)
{
    GTM_TRY(check_sizes("gtm_embed_gradient", type, rows, columns, number_of_ids, number_of_bags));
    if (!table_gradient || (number_of_ids && (!offsets || number_of_bags) && (!ids || !gradient))) return fail(GTM_ERR_ARG, "gtm_embed_gradient: null array");
    if ((uintptr_t)gradient % type_bytes(type) || (uintptr_t)ids % (ids_64 ? 8 : 4) || (uintptr_t)offsets % (offsets_64 ? 8 : 4))
        return fail(GTM_ERR_ARG, "gtm_embed_gradient: an array does not start at a boundary of its elements");
    if (gradient_stride < 0 || gradient_stride >= kMostRows) return fail(GTM_ERR_ARG, "gtm_embed_gradient: row stride %lld of the gradient", (long long)gradient_stride);
    if ((uintptr_t)table_gradient % 16) return fail(GTM_ERR_ARG, "gtm_embed_gradient: the result does not start at a 16-byte boundary");
    const long long n = offsets && number_of_bags == 0 ? 0 : number_of_ids;          // no bag, no id
    const GradientSpace space = gradient_space(n, rows, columns);
    if (workspace_bytes < space.total || !workspace || (uintptr_t)workspace % 16)
        return fail(GTM_ERR_ARG, "gtm_embed_gradient: workspace of %llu bytes, %llu needed (16-byte aligned)", (unsigned long long)workspace_bytes, (unsigned long long)space.total);
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    char *w = (char *)workspace;
    uint2 *from = (uint2 *)(w + space.pairs[0]), *to = (uint2 *)(w + space.pairs[1]);
    unsigned *counts = (unsigned *)(w + space.counts);
    if (n) {
        const unsigned tiles = (unsigned)space.tiles;
        const auto sort = [&](auto each) -> int {
            constexpr int kEach = decltype(each)::value;
            GTM_TRY(launch_early(sort_keys_kernel<kEach>, dim3(tiles), dim3(kSortThreads), 0, stream, ids, ids_64, n, offsets, offsets_64, (long long)number_of_bags, (unsigned)rows, from, counts));
            for (int shift = 0; shift < 32 && ((uint64_t)rows >> shift) != 0; shift += kDigit) {
                if (shift) GTM_TRY(launch_early(sort_count_kernel<kEach>, dim3(tiles), dim3(kSortThreads), 0, stream, from, n, shift, counts));
                GTM_TRY(launch_early(sort_scan_kernel, dim3(1), dim3(1024), 0, stream, counts, (int)tiles));
                GTM_TRY(launch_early(sort_place_kernel<kEach>, dim3(tiles), dim3(kSortThreads), 0, stream, from, n, shift, counts, to));
                std::swap(from, to);
            }
            return GTM_OK;
        };
        GTM_TRY(space.each == 4 ? sort(std::integral_constant<int, 4>()) : sort(std::integral_constant<int, 16>()));
    }
    GTM_TRY(launch_early(sort_rows_kernel, dim3((unsigned)((n + 256) / 256)), dim3(256), 0, stream, from, n, (long long)rows, (int *)(w + space.offsets)));
    GatherArgs a;
    a.src = gradient, a.src_stride = gradient_stride, a.rows = offsets ? number_of_bags : n;
    a.pairs = from, a.list = nullptr, a.list_wide = 0, a.positions = n;
    a.offsets = w + space.offsets, a.offsets_wide = 0, a.segments = rows;
    a.columns = (int)columns, a.scale = scale, a.out = table_gradient, a.out_stride = columns;
    return launch_gather(a, type, w, space.gather, stream);
}
