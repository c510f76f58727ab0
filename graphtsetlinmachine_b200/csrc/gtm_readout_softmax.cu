// Softmax cross entropy over many labels, its gradient, and the most probable label.
//
//   l[n, v] = scale * x[n] . w[v]        lse[n] = log sum_v exp l[n, v]        loss[n] = lse[n] - l[n, label[n]]
//   P = (softmax(l) - onehot(label)) * gradient[n] * scale        dx = P w        dw = P^T x
//
// The logits are never kept.  Forward, a tile of them stays in tensor memory and leaves the largest value and the sum of exponentials of
// every row, which a second kernel joins.  Backward, the labels are taken in pieces: a piece's logits are computed again, P of
// the piece goes to the workspace in the operands' 16-bit type, and two products use it.  All products are one kernel on
// tcgen05 over pairs of thread blocks: tiles of 256 x 256 (or 128), operands by TMA through a ring in shared memory, sums in tensor
// memory, two tiles deep, so that a tile's epilogue runs under the next tile's products; results leave by TMA too.  dw and dx of a piece are one
// launch: dw's tiles go round, and dx's work fills up what is left of the last round.  For up to two examples (eight in 32 bits) the prediction
// is a kernel of plain dot products, whose time is that of reading w.  The loss of so few stays with the product kernel: the gradient takes
// P from the same logits then, and where P of the label is near one, a logit's error leaves it with the normaliser.
//
// 16-bit inputs are multiplied as they are, with sums in 32 bits.  32-bit inputs are split into three bf16 parts (24 bits of fraction),
// and the six products of parts that reach 2^-24 are added, the smallest first.  The tensor cores cut sums off instead of rounding them, about 3e-8 of
// the sum at every step of 16 elements (1e-7 where all terms have one sign) and always towards zero.  So logits are summed in chunks of up to 320 elements (128 of inputs
// of 32 bits), which the epilogue adds up in registers, with rounding; and sums for dw and dx of 32-bit inputs go to memory after 512
// elements, where they are added with rounding.  P is rounded to the operands' type, to as many bits as
// dx and dw are (their errors are 1.25 times as large for it on the median of 78 problems, twice for a single example, whose P are all of a sum; P in two parts would
// double both products); fp16 has too small a range for that, so P is scaled by 2^14 over the largest finite |gradient * scale| there (2^-38 of that is the smallest
// step of P: an example that weighs 2^-20 of another has fewer bits).
#include "gtm_readout.cuh"
#include "gtm_readout_mma.cuh"
#include "gtm_readout_softmax.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace gtm_readout {
namespace {

constexpr int kDepth = 64;                                 // elements of a sum's index per stage of the ring
constexpr int kHalfBytes = 128 * kDepth * 2;               // an operand's share of a stage in one thread block
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kThreads = 384, kEpilogue = 8;               // warps 0: copies, 1: products, 2: tensor memory; 4..11: epilogue
constexpr int kBoxBytes = 32 * 128;                        // 32 rows of 128 bytes: what a warp of the epilogue stores at once, from two buffers in turn
// Registers of a thread: as many as launched with (kLaunchedRegisters, the most for so many threads) are split anew between the first four warps and the epilogue, which holds 128 logits.
constexpr int kLaunchedRegisters = 168, kFewRegisters = 104, kManyRegisters = 200;
static_assert(128 * kFewRegisters + (kThreads - 128) * kManyRegisters <= kThreads * kLaunchedRegisters, "a block waits for registers that it does not have");
constexpr int kPairs = 74;                                 // pairs of SMs
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kPieceBytes = 128 << 20;                 // of P in the workspace at a time
constexpr int64_t kStatBytes = 64 << 20;                   // of partial sums of exponentials at a time
constexpr int kLongestSum = 512;                           // blocks of a sum in tensor memory, for gradients of 16 bits: 2,048 steps cut off up to 2e-4 of it

enum Epilogue { kSums = 0, kBest = 1, kProb = 2, kOut = 3 };
__host__ __device__ constexpr int stages_of(int mode) { return mode == kSums || mode == kBest ? 6 : 5; }
__host__ __device__ constexpr size_t shared_of(int mode) { return 1024 + stages_of(mode) * kStageBytes + (mode == kSums || mode == kBest ? 0 : kEpilogue * 2 * kBoxBytes); }

// Parts of a 32-bit operand that are multiplied, the smallest products first: pairs (a, b) of two bits each.
constexpr int kPartProducts = 6;
__device__ __forceinline__ void parts_of(int products, int i, int &a, int &b)
{
    constexpr unsigned as = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10, bs = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;
    a = products == 1 ? 0 : as >> (2 * i) & 3;
    b = products == 1 ? 0 : bs >> (2 * i) & 3;
}

// One product.  Its work is tiles of 256 rows over blocks of the sum's index (`blocks` of kDepth each, times products of parts).
struct Product {
    long long rows, columns;                    // of the result
    int m_tiles, n_tiles, tile_columns;         // 256 or 128 columns of a tile
    int m_fast;                                 // tiles of one column block follow each other
    int depth_blocks, products, blocks, per_split;  // blocks of a tile are cut into splits of per_split
    int chunk;                                  // blocks of the index whose products of parts follow each other; sums of several products end with them
    int a_rows;                                 // operand A's rows, not the sum's index, lie next to each other (operand B's never do: that is a third slower)
    int a_first;                                // offset of the sum's index in operand A (a row of W)
    int b_row;                                  // offset of the result's columns in operand B (a row of W)
    unsigned what;                              // instruction descriptor
    int add;                                    // the result is added to what is there
    int type;                                   // of the result: GTM_F32 (slices of sums too) or a 16-bit type
    const unsigned *out_scale;                  // bits of the largest finite |factor|: the result is 2^-14 times this, null: 1

    __host__ __device__ int tiles() const { return m_tiles * n_tiles; }
    __host__ __device__ int splits() const { return (blocks + per_split - 1) / per_split; }
    __host__ __device__ void tile(int t, int &m, int &n) const
    {
        if (m_fast) m = t % m_tiles, n = t / m_tiles;
        else n = t % n_tiles, m = t / n_tiles;
    }
};

// Who does what: the splits of the first product's tiles go to the pairs of SMs in turn; the blocks of the second one's tiles, in a row, are cut so
// that all pairs end together, wherever in a tile that is.  The pieces of a tile are slices of sums, added up later.  A pair begins with the second product, whose
// results are the larger ones: they leave while it works on the first.
struct Schedule {
    int items, pairs, longer;                   // of the first product; pairs that have one item more
    int others;                                 // pairs behind those that share the rest of the second product's blocks
    long long units, units_of_longer;           // blocks of the second product; of these, the share of the longer pairs

    __host__ __device__ long long begin(int pair) const
    {
        if (pair <= longer) return longer ? units_of_longer * pair / longer : 0;
        const int at = pair - longer < others ? pair - longer : others;
        return units_of_longer + (units - units_of_longer) * at / others;
    }
    __host__ __device__ int pair_of(long long unit) const
    {
        int i = unit < units_of_longer ? (int)(unit * longer / units_of_longer) : longer + (int)((unit - units_of_longer) * others / (units - units_of_longer));
        while (i > 0 && begin(i) > unit) i--;
        while (i + 1 < pairs && begin(i + 1) <= unit) i++;
        return i;
    }
    __host__ __device__ int slices(long long blocks, int tile) const { return pair_of((tile + 1) * blocks - 1) - pair_of(tile * blocks) + 1; }
};

// Tensor maps are the launch's own arguments; the second product's are used in kOut alone.
struct Maps {
    CUtensorMap a[2], b[2], out[2];
};

struct Launch {
    Product p[2];
    Schedule schedule;
    unsigned *error;                            // counts waits that ran out
    unsigned long long limit;                   // of a wait, nanoseconds
    int lost;                                   // copies are left out, so that waits run out
    // kSums, kBest
    float2 *sums;                               // [part][rows]: largest product and sum of exponentials (kBest: all but the largest's)
    int *best;                                  // [part][rows]
    float *label_logit;                         // [rows], products
    float scale;
    // kSums, kProb
    const int *labels;                          // -1: none
    int first_label;                            // label of column 0
    // kProb
    const float *normalisers, *factors;         // [rows]
    const unsigned *largest;                    // bits of the largest finite |factor|, null: factors as they are
};

// A pair's work, piece by piece.
template <bool kCut>
struct Work {
    const Launch &l;
    int pair, item, at;                          // the next item of the first product, and where in it
    long long unit, begin, end;
    // the piece at hand: product, tile, blocks [first, last), whether its sums are the first of their tile and slice
    int which, m, n, first, last, split;
    bool fresh;

    __device__ __forceinline__ explicit Work(const Launch &launch) : l(launch)
    {
        pair = blockIdx.x / 2, item = pair, at = 0;
        unit = begin = l.schedule.units ? l.schedule.begin(pair) : 0;
        end = l.schedule.units ? l.schedule.begin(pair + 1) : 0;
    }
    // The end of a piece that begins at block `from`: of sums in memory a chunk (of several products of parts), of logits the tile.
    __device__ __forceinline__ static int cut(const Product &p, int from, long long end)
    {
        if (!kCut) return p.blocks;
        const int chunk = p.chunk * p.products;
        return (int)min(end, p.products == 1 ? (long long)p.blocks : min((long long)p.blocks, (from / chunk + 1ll) * chunk));
    }
    __device__ __forceinline__ bool next()
    {
        if (unit < end) {
            which = 1;
            const Product &p = l.p[1];
            const int tile = (int)(unit / p.blocks);
            p.tile(tile, m, n);
            first = (int)(unit - (long long)tile * p.blocks), last = cut(p, first, first + end - unit);
            fresh = first == 0 || unit == begin;
            split = tile;                        // its slice is looked up by who needs it
            unit += last - first;
            return true;
        }
        if (item >= l.schedule.items) return false;
        which = 0;
        const Product &p = l.p[0];
        split = item / p.tiles();
        p.tile(item - split * p.tiles(), m, n);
        const int from = split * p.per_split, to = min(p.blocks, from + p.per_split);
        first = from + at, last = cut(p, first, to);
        fresh = at == 0;
        at += last - first;
        if (last == to) item += l.schedule.pairs, at = 0;
        return true;
    }
    __device__ __forceinline__ int slice() const { return which == 0 ? split : pair - l.schedule.pair_of((long long)split * l.p[1].blocks); }
};

// Of exponents of two.  A scale may be so large that this would be infinite, and infinity times the distance zero no number.
__device__ __forceinline__ float slope_of(float scale) { return fminf(scale * kLog2e, 3.402823466e38f); }

// Softmax statistics of a row, over some of its products at a time.
struct RowSums {
    float largest, sum;
    __device__ __forceinline__ static RowSums none() { return {-INFINITY, 0.f}; }
    template <int N>
    __device__ __forceinline__ void take(const float (&v)[N], float slope)
    {
        float top = v[0];
#pragma unroll
        for (int j = 1; j < N; j++) top = fmaxf(top, v[j]);
        const float next = fmaxf(largest, top), from = next == -INFINITY ? 0.f : next;
        if (largest > -INFINITY) sum *= exp2_fast((largest - from) * slope);
#pragma unroll
        for (int j = 0; j < N; j++) sum += exp2_fast((v[j] - from) * slope);
        largest = next;
    }
};

// The same with the first largest one's index and without its own 1 in the sum.
struct RowBest {
    float largest, rest;
    int index;
    __device__ __forceinline__ static RowBest none() { return {-INFINITY, 0.f, -1}; }
    template <int N>
    __device__ __forceinline__ void take(const float (&v)[N], float slope, int first)
    {
        float top = v[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < N; j++)
            if (v[j] > top || !(top == top)) top = v[j], at = j;
        const float from = top == -INFINITY || !(top == top) ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) sum += j == at && top > -INFINITY ? 0.f : exp2_fast((v[j] - from) * slope);
        add(top, sum, slope, first + at);
    }
    __device__ __forceinline__ void add(float top, float sum, float slope, int at)
    {
        if (!(top > -INFINITY)) rest += sum;                       // nothing but -inf (sum is 0) or NaN
        else if (top > largest) rest = (largest > -INFINITY ? (rest + 1.f) * exp2_fast((largest - top) * slope) : rest) + sum, largest = top, index = at;
        else rest += (sum + 1.f) * exp2_fast((top - largest) * slope);
    }
};

// A warp's boxes on their way to memory: written to one of two buffers, rows of 128 bytes swizzled as the map says, and stored from there.
struct BoxStore {
    unsigned buffers;
    int turn = 0;
    // 16-byte piece `j` (of 8) of the lane's row
    __device__ __forceinline__ void put(int j, uint4 v) const
    {
        const unsigned lane = threadIdx.x & 31;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buffers + turn * kBoxBytes + lane * 128 + ((j ^ (lane & 7)) * 16)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
    // The buffer whose turn it is has been read.
    __device__ __forceinline__ void begin() const
    {
        if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void send(const CUtensorMap *map, int x, int y, int z, bool add)
    {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            if (add) asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(buffers + turn * kBoxBytes), "r"(x), "r"(y), "r"(z) : "memory");
            else asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(buffers + turn * kBoxBytes), "r"(x), "r"(y), "r"(z) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        turn ^= 1;
    }
    __device__ __forceinline__ static void finish()
    {
        if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
};

__device__ __forceinline__ unsigned pack2(float a, float b, bool fp16)
{
    if (fp16) {
        const __half2 h = __floats2half2_rn(a, b);
        return reinterpret_cast<const unsigned &>(h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const unsigned &>(h);
}

// 64 columns of 16 bits: one box.
__device__ __forceinline__ void send_16(BoxStore &to, const float (&v)[64], bool fp16, const CUtensorMap *map, int x, int y, int z)
{
    to.begin();
#pragma unroll
    for (int j = 0; j < 8; j++)
        to.put(j, make_uint4(pack2(v[j * 8], v[j * 8 + 1], fp16), pack2(v[j * 8 + 2], v[j * 8 + 3], fp16), pack2(v[j * 8 + 4], v[j * 8 + 5], fp16), pack2(v[j * 8 + 6], v[j * 8 + 7], fp16)));
    to.send(map, x, y, z, false);
}

// 64 columns of 32 bits: two boxes, the second only where there are columns for it.
__device__ __forceinline__ void send_32(BoxStore &to, const float (&v)[64], const CUtensorMap *map, int x, int y, int z, bool add, long long left)
{
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (left <= h * 32) break;
        to.begin();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float *q = v + h * 32 + j * 4;
            to.put(j, make_uint4(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3])));
        }
        to.send(map, x + h * 32, y, z, add);
    }
}

// The product kernel.  A pair of blocks has a tile of 256 x 256: each loads its 128 rows of A and half of B, 32 KB for 64 elements of the sum's index, which
// the tensor cores take 512 cycles for and shared memory, at 128 bytes a cycle written and read once, as long: both are at their limit, as is, in longer runs, the
// GPU's power.  A block of 64 takes 0.42 to 0.46 us.  Of 8,192 x 1,024 features and 65,536 labels: statistics 0.83 to 1.02 ms (1.1 to 1.3 PFLOP/s by
// the clock that the power leaves), P 1.24 to 1.35 ms, both gradients 1.85 to 1.99 ms (1.1 to 1.2).  A commit takes 120 cycles of the tensor cores.  A sixth stage of the ring, or a seventh, changed nothing.
template <int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) softmax_product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Launch l)
{
    constexpr int kStages = stages_of(kMode);
    constexpr bool kStores = kMode == kProb || kMode == kOut;
    extern __shared__ unsigned char shared_raw[];
    __shared__ alignas(8) unsigned long long barriers[2 * kStages + 4];
    __shared__ unsigned tmem_shared;
    const unsigned ring = (smem_address(shared_raw) + 1023) & ~1023u;
    const unsigned full = smem_address(barriers), empty = full + 8 * kStages, sums_full = empty + 8 * kStages, sums_empty = sums_full + 16;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const unsigned rank = cluster_rank();
    next_may_start();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) barrier_init(full + 8 * i, 1), barrier_init(empty + 8 * i, 1);
        for (int i = 0; i < 2; i++) barrier_init(sums_full + 8 * i, 1), barrier_init(sums_empty + 8 * i, 2 * kEpilogue);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_allocate(smem_address(&tmem_shared), 512);
    __syncthreads();
    tmem_before_sync();
    cluster_sync();
    tmem_after_sync();
    const unsigned tmem = tmem_shared;
    wait_for_previous();

    bool fine = true;
    if (warp < 4) {
        if constexpr (kMode != kOut) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
        if (warp == 0 && lane == 0) {
            // copies: the ring's stages of this block, counted on the leader's barriers
            int stage = 0, phase = 0;
            for (Work<kMode == kOut> w(l); fine && !l.lost && w.next();) {
                const Product &p = l.p[w.which];
                const CUtensorMap *map_a = &maps.a[w.which], *map_b = &maps.b[w.which];
                const int half_columns = p.tile_columns / 2;
                const int m0 = w.m * 256 + (int)rank * 128, n0 = w.n * p.tile_columns + (int)rank * half_columns + p.b_row;
                // the product of parts, and the block of the sum's index, of a chunk at a time
                int chunk_first = w.first == 0 ? 0 : w.first / (p.chunk * p.products) * p.chunk, chunk_blocks = min(p.chunk, p.depth_blocks - chunk_first);
                int product = w.first == 0 ? 0 : (w.first - chunk_first * p.products) / chunk_blocks, block = w.first - chunk_first * p.products - product * chunk_blocks;
                for (int i = w.first; i < w.last; i++) {
                    if (!(fine = barrier_wait(empty + 8 * stage, phase ^ 1, l.limit))) break;
                    const unsigned to = ring + stage * kStageBytes, bar = in_leader(full + 8 * stage);
                    if (rank == 0) barrier_expect(full + 8 * stage, 2 * (kHalfBytes + half_columns * kDepth * 2));
                    int part_a, part_b;
                    parts_of(p.products, product, part_a, part_b);
                    const int k = (chunk_first + block) * kDepth;
                    if (p.a_rows)
                        for (int g = 0; g < 2; g++) load_box(map_a, to + g * 8192, bar, m0 + g * 64, p.a_first + k, part_a);
                    else load_box(map_a, to, bar, k, m0, part_a);
                    load_box(map_b, to + kHalfBytes, bar, k, n0, part_b);
                    if (++block == chunk_blocks) {
                        block = 0;
                        if (++product == p.products) product = 0, chunk_first += chunk_blocks, chunk_blocks = min(p.chunk, p.depth_blocks - chunk_first);
                    }
                    if (++stage == kStages) stage = 0, phase ^= 1;
                }
            }
            // the products' last arrivals come to this block's barriers before it ends
            for (int i = 0; i < kStages && fine; i++) {
                fine = barrier_wait(empty + 8 * stage, phase ^ 1, l.limit);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
            // copies that nobody will wait for any more end before the block does: 20 ms are thousands of times what one takes
            if (!fine)
                for (const unsigned long long began = nanoseconds(); nanoseconds() - began < 20000000ull;) __nanosleep(1000);
        } else if (warp == 1 && lane == 0 && rank == 0) {
            // barriers of the next stage and of the next sum are asked before products are issued, and answer while they are
            int stage = 0, phase = 0, buffer = 0, buffer_phase = 0;
            bool loaded = false, drained = true;
            for (Work<kMode == kOut> w(l); fine && w.next();) {
                const Product &p = l.p[w.which];
                // rows next to each other: 64 of them and 8 of the sum's index are 1024 bytes, 64 more rows one box further; a step of 16 is 2048 bytes.
                // the sum's index next to each other: 8 rows are 1024 bytes; a step of 16 is 32 bytes
                const unsigned a_leading = p.a_rows ? 8192 : 16, a_step = p.a_rows ? 2048 : 32, what = p.what;
                const int chunk = kMode == kOut ? w.last - w.first : p.chunk * p.products;
                for (int first = w.first; fine && first < w.last; first += chunk) {
                    const unsigned to = tmem + buffer * 256, sums = sums_full + 8 * buffer;
                    if (!drained && !(fine = barrier_wait(sums_empty + 8 * buffer, buffer_phase ^ 1, l.limit))) break;
                    if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
                    const int blocks = min(chunk, w.last - first);
                    for (int i = 0; i < blocks; i++) {
                        if (!loaded && !(fine = barrier_wait(full + 8 * stage, phase, l.limit))) break;
                        tmem_after_sync();
                        const unsigned a = ring + stage * kStageBytes, b = a + kHalfBytes, done = empty + 8 * stage;
                        if (++stage == kStages) stage = 0, phase ^= 1;
                        loaded = barrier_test(full + 8 * stage, phase);
                        drained = barrier_test(sums_empty + 8 * buffer, buffer_phase ^ 1);
#pragma unroll
                        for (int k = 0; k < kDepth / 16; k++)
                            multiply(to, operand(a + k * a_step, a_leading, 1024), operand(b + k * 32, 16, 1024), what, i > 0 || k > 0);
                        commit_to_pair(done);
                    }
                    if (fine) commit_to_pair(sums);
                }
            }
        }
    } else {
        if constexpr (kMode != kOut) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
        const int quarter = (warp - 4) & 3, half = (warp - 4) / 4;
        int buffer = 0, buffer_phase = 0;
        BoxStore store = {ring + kStages * kStageBytes + (warp - 4) * 2 * kBoxBytes};
        for (Work<kMode == kOut> w(l); w.next();) {
            const Product &p = l.p[w.which];
            const int half_columns = p.tile_columns / 2;
            const long long row0 = (long long)w.m * 256 + rank * 128 + quarter * 32, row = row0 + lane;
            const bool real = row < p.rows;
            const long long column0 = (long long)w.n * p.tile_columns + half * half_columns;
            const unsigned tile = tmem + half * half_columns + ((unsigned)(quarter * 32) << 16);
            // Whichever wait of the pair runs out, this one does too.  What was not multiplied is NaN then, in this tile and in those that are to come
            const auto arrived = [&] {
                if (fine) fine = __all_sync(~0u, barrier_wait(sums_full + 8 * buffer, buffer_phase, l.limit));
                if (fine) tmem_after_sync();
                return fine;
            };
            const auto leave = [&] {
                // the tile's last columns are in registers: the next but one may overwrite it
                tmem_before_sync();
                __syncwarp();
                if (lane == 0) barrier_arrive_leader(in_leader(sums_empty + 8 * buffer));
                if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
            };
            if constexpr (kMode == kOut) {
                const int slice = w.slice();
                const float out_scale = p.out_scale ? __uint_as_float(*p.out_scale) * (1.f / 16384.f) : 1.f;
                arrived();
#pragma unroll 1
                for (int c = 0; c < half_columns; c += 64) {
                    const long long column = column0 + c, left = p.columns - column;
                    if (left <= 0) break;                                   // the warp together
                    float v[64];
                    if (fine) {
                        tmem_load64(tile + buffer * 256 + c, v);
                        if (c + 64 >= half_columns || left <= 64) leave();
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; j++) v[j] = __int_as_float(0x7fffffff);
                    }
#pragma unroll
                    for (int j = 0; j < 64; j++) v[j] *= out_scale;
                    if (row0 >= p.rows) continue;
                    // what is added to has to be there, or the order of two additions would be open
                    if (p.products > 1 && !w.fresh) BoxStore::finish();
                    if (p.type == GTM_F32) send_32(store, v, &maps.out[w.which], (int)column, (int)row0, slice, p.add || !w.fresh, left);
                    else send_16(store, v, p.type == GTM_F16, &maps.out[w.which], (int)column, (int)row0, slice);
                }
                if (fine && column0 >= p.columns) leave();                  // no column of this half
            } else {
                float normaliser = 0.f, factor = 0.f;
                int label = -1;
                if ((kMode == kSums || kMode == kProb) && real && l.labels) label = l.labels[row] - l.first_label;
                if (kMode == kProb && real) {
                    normaliser = l.normalisers[row], factor = l.factors[row];
                    if (l.largest) {
                        // a factor that is not finite has no part in the largest: it is its example's alone
                        factor = factor == 0.f ? 0.f : isfinite(factor) ? factor / __uint_as_float(*l.largest) * 16384.f : __int_as_float(0x7fffffff);
                    }
                }
                float sum[128];                   // a tile's logits of the lane's row, added up chunk by chunk
                for (int done = 0; done < p.depth_blocks; done += p.chunk) {
                    if (!arrived()) break;
                    const unsigned from = tile + buffer * 256;
#pragma unroll
                    for (int c = 0; c < 128; c += 32) {
                        if (c >= half_columns || column0 + c >= p.columns) break;
                        if (done == 0) {
                            tmem_load32(from + c, reinterpret_cast<float (&)[32]>(sum[c]));
                        } else {
                            float more[32];
                            tmem_load32(from + c, more);
#pragma unroll
                            for (int j = 0; j < 32; j++) sum[c + j] += more[j];
                        }
                    }
                    leave();
                }
                if (!fine)
#pragma unroll
                    for (int j = 0; j < 128; j++) sum[j] = __int_as_float(0x7fffffff);
                RowSums sums = RowSums::none();
                RowBest best = RowBest::none();
#pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    const long long column = column0 + c, left = p.columns - column;
                    if (c >= half_columns || left <= 0) break;              // the warp together
                    float (&v)[64] = reinterpret_cast<float (&)[64]>(sum[c]);
                    if (kMode == kSums || kMode == kBest) {
                        if (left < 64)
#pragma unroll
                            for (int j = 0; j < 64; j++)
                                if (j >= left) v[j] = -INFINITY;
                        if (kMode == kSums) {
                            sums.take(v, slope_of(l.scale));
                            const long long at = label - column;
                            if (__any_sync(~0u, at >= 0 && at < 64 && label >= 0)) {
                                float mine = 0.f;
#pragma unroll
                                for (int j = 0; j < 64; j++)
                                    if (at == j) mine = v[j];
                                if (label >= 0 && at >= 0 && at < 64 && real) l.label_logit[row] = mine;
                            }
                        } else {
                            best.take(v, slope_of(l.scale), (int)column);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; j++) v[j] = exp2_fast(fmaf(v[j], l.scale, -normaliser) * kLog2e);
                        const long long at = label - column;
                        if (__any_sync(~0u, at >= 0 && at < 64))
#pragma unroll
                            for (int j = 0; j < 64; j++)
                                if (at == j) v[j] -= 1.f;
#pragma unroll
                        for (int j = 0; j < 64; j++) v[j] = factor == 0.f ? 0.f : v[j] * factor;
                        if (row0 >= p.rows) continue;                       // the warp together
                        send_16(store, v, p.type == GTM_F16, &maps.out[0], (int)column, (int)row0, 0);
                        if (p.products > 1)
#pragma unroll 1
                            for (int part = 1; part < 3; part++) {
#pragma unroll
                                for (int j = 0; j < 64; j++) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
                                send_16(store, v, false, &maps.out[0], (int)column, (int)row0, part);
                            }
                    }
                }
                if ((kMode == kSums || kMode == kBest) && real) {
                    const long long at = (w.n * 2ll + half) * p.rows + row;
                    l.sums[at] = kMode == kSums ? make_float2(sums.largest, sums.sum) : make_float2(best.largest, best.rest);
                    if (kMode == kBest) l.best[at] = best.index;
                }
            }
        }
        if (kStores) BoxStore::finish();
    }
    if (!fine && lane == 0) atomicAdd(l.error, 1u);
    __syncwarp();
    tmem_before_sync();
    cluster_sync();
    tmem_after_sync();
    if (warp == 2) tmem_free(tmem, 512);
}

// The prediction for few examples, whose time is that of reading the weights.  A whole pass over 131,072 x 1,024 bf16 takes 51 us for one example
// (5.3 TB/s), 58 for two and 90 for four; with the product kernel, most of its rows being outside of the matrix, it takes 74 to 80 for any of them.  Dot products
// in 32 bits, four rows of weights in a warp at a time (two, and twice the blocks, where the sums of several examples take the registers: 82 us for two
// examples with four), of every lane 16 bytes (or, where rows start anywhere, an element).  A lane keeps the statistics of one of the rows' products with
// one example; a block leaves one part.
constexpr int kFewThreads = 256;
__host__ __device__ constexpr int few_rows(size_t element, int examples) { return element == 2 && examples > 1 ? 2 : 4; }

struct FewArgs {
    const void *x, *w;
    long long x_stride, w_stride;
    int examples, labels, columns;
    float scale;
    float2 *sums;
    int *best;
};

template <class T, int kExamples, bool kWhole>
__global__ void __launch_bounds__(kFewThreads) softmax_few_kernel(const FewArgs a)
{
    next_may_start();
    wait_for_previous();
    constexpr int V = kWhole ? 16 / sizeof(T) : 1, kRows = few_rows(sizeof(T), kExamples), kValues = kExamples * kRows, kStep = 32 * V, kUnroll = sizeof(T) == 2 ? 4 : 2;
    extern __shared__ float4 shared_x4[];
    float *shared_x = (float *)shared_x4;       // [example][columns, rounded up to the step]
    __shared__ RowBest block_best[kFewThreads / 32][kValues];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, padded = (a.columns + kStep - 1) / kStep * kStep;
    for (int i = threadIdx.x; i < kExamples * padded; i += kFewThreads) {
        const int e = i / padded, c = i - e * padded;
        shared_x[i] = e < a.examples && c < a.columns ? to_float(((const T *)a.x)[e * a.x_stride + c]) : 0.f;
    }
    __syncthreads();
    RowBest best = RowBest::none();
    const int my_row = lane / kExamples;        // lanes behind kValues keep nothing
    for (long long v0 = ((long long)blockIdx.x * (kFewThreads / 32) + warp) * kRows; v0 < a.labels; v0 += (long long)gridDim.x * (kFewThreads / 32) * kRows) {
        float dot[kRows][kExamples];
        const T *row[kRows];
#pragma unroll
        for (int r = 0; r < kRows; r++) {
            row[r] = (const T *)a.w + min(v0 + r, (long long)a.labels - 1) * a.w_stride;
#pragma unroll
            for (int e = 0; e < kExamples; e++) dot[r][e] = 0.f;
        }
#pragma unroll kUnroll
        for (int c0 = 0; c0 < a.columns; c0 += kStep) {
            const int c = c0 + lane * V;
            Pack<T, V> w[kRows];
#pragma unroll
            for (int r = 0; r < kRows; r++)
                if (c < a.columns) w[r] = *(const Pack<T, V> *)(row[r] + c);
                else
#pragma unroll
                    for (int i = 0; i < V; i++) w[r].v[i] = from_float<T>(0.f);
#pragma unroll
            for (int e = 0; e < kExamples; e++) {
                float x[V];
                if constexpr (kWhole)
#pragma unroll
                    for (int i = 0; i < V; i += 4) reinterpret_cast<float4 &>(x[i]) = *(const float4 *)(shared_x + e * padded + c + i);
                else x[0] = shared_x[e * padded + c];
#pragma unroll
                for (int r = 0; r < kRows; r++)
#pragma unroll
                    for (int i = 0; i < V; i++) dot[r][e] = fmaf(to_float(w[r].v[i]), x[i], dot[r][e]);
            }
        }
        float mine = 0.f;
#pragma unroll
        for (int r = 0; r < kRows; r++)
#pragma unroll
            for (int e = 0; e < kExamples; e++) {
#pragma unroll
                for (int o = 16; o; o /= 2) dot[r][e] += __shfl_xor_sync(~0u, dot[r][e], o);
                if (lane == r * kExamples + e) mine = dot[r][e];
            }
        if (lane < kValues && v0 + my_row < a.labels) {
            const float one[1] = {mine};
            best.take(one, slope_of(a.scale), (int)(v0 + my_row));
        }
    }
    if (lane < kValues) block_best[warp][lane] = best;
    __syncthreads();
    if (threadIdx.x >= kExamples || threadIdx.x >= a.examples) return;
    const float slope = slope_of(a.scale);
    RowBest top = RowBest::none();
    for (int w = 0; w < kFewThreads / 32; w++)
        for (int r = 0; r < kRows; r++) {
            const RowBest b = block_best[w][r * kExamples + threadIdx.x];
            // labels of different warps are in no order: of equal products the lower label is the best
            const bool lower = b.largest == top.largest && b.index < top.index;
            const int index = b.index;
            top.add(b.largest, b.rest, slope, index);
            if (lower && b.largest > -INFINITY) top.index = index;
        }
    const long long at = (long long)blockIdx.x * a.examples + threadIdx.x;
    a.sums[at] = make_float2(top.largest, top.rest);
    a.best[at] = top.index;
}

// ------------------------------------------------------------------------------------------- around the products
// The next part of a 32-bit value, of which the rest is left: rounded, and towards zero where rounding would leave the range (the lowest value, with which
// labels are masked, has to stay finite: an infinite part times a part that is zero is no number).
__device__ __forceinline__ __nv_bfloat16 part_of(float &rest)
{
    __nv_bfloat16 part = __float2bfloat16_rn(rest);
    if (isinf(__bfloat162float(part)) && !isinf(rest)) part = __float2bfloat16_rz(rest);
    const float held = __bfloat162float(part);
    rest = isfinite(held) ? rest - held : 0.f;
    return part;
}

// Rows of a matrix with 16-byte boundaries, in parts where they are 32-bit ones; rows of examples that are ignored are zero.  A thread has eight
// elements in a row; kWhole: rows start at 16-byte boundaries and have all eight.
template <class T, bool kWhole>
__global__ void __launch_bounds__(256) softmax_lay_out_kernel(const T *from, long long stride, long long rows, int columns, const int *labels, __nv_bfloat16 *to, long long to_stride, long long part)
{
    next_may_start();
    wait_for_previous();
    constexpr int kWide = 16 / sizeof(T);
    const int per_row = (columns + 7) / 8;
    const long long all = rows * per_row;
    const bool narrow = all < 1ll << 32;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long r = narrow ? (long long)((unsigned)i / (unsigned)per_row) : i / per_row;
        const int c = (int)(i - r * per_row) * 8;
        const bool kept = !labels || labels[r] != -1;
        Pack<T, 8> v;
        if (kWhole && kept) {
#pragma unroll
            for (int k = 0; k < 8; k += kWide) reinterpret_cast<Pack<T, kWide> &>(v.v[k]) = *(const Pack<T, kWide> *)(from + r * stride + c + k);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v.v[k] = kept && c + k < columns ? from[r * stride + c + k] : from_float<T>(0.f);
        }
        // the copy's rows have room up to a multiple of eight
        __nv_bfloat16 *q = to + r * to_stride + c;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int p = 0; p < 3; p++) {
                Pack<__nv_bfloat16, 8> b;
#pragma unroll
                for (int k = 0; k < 8; k++) b.v[k] = part_of(v.v[k]);
                *(Pack<__nv_bfloat16, 8> *)(q + p * part) = b;
            }
        } else {
            *(Pack<T, 8> *)q = v;
        }
    }
}

// The gradient's x: rows as above, and the same matrix with rows for columns, which dw's product takes.  A block has 64 rows and 64 columns.
template <class T>
__global__ void __launch_bounds__(256) softmax_lay_out_both_kernel(const T *from, long long stride, long long rows, int columns, const int *labels, __nv_bfloat16 *to, long long to_stride, long long part,
                                                                   __nv_bfloat16 *turned, long long turned_stride, long long turned_part, bool whole)
{
    next_may_start();
    wait_for_previous();
    using Out = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;
    constexpr int kParts = sizeof(T) == 4 ? 3 : 1, kWide = 16 / sizeof(T);
    __shared__ Out tile[kParts][64][72];                      // rows of 144 bytes: eight of them read as columns meet different banks
    const long long row0 = (long long)blockIdx.x * 64;
    const int column0 = blockIdx.y * 64, c8 = threadIdx.x % 8 * 8, r0 = threadIdx.x / 8;
#pragma unroll
    for (int h = 0; h < 64; h += 32) {
        const long long r = row0 + r0 + h;
        const int c = column0 + c8;
        const bool kept = r < rows && (!labels || labels[r] != -1);
        Pack<T, 8> v;
        if (whole && kept && c < columns) {
#pragma unroll
            for (int k = 0; k < 8; k += kWide) reinterpret_cast<Pack<T, kWide> &>(v.v[k]) = *(const Pack<T, kWide> *)(from + r * stride + c + k);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v.v[k] = kept && c + k < columns ? from[r * stride + c + k] : from_float<T>(0.f);
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            Pack<Out, 8> b;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if constexpr (kParts == 1) b.v[k] = v.v[k];
                else b.v[k] = part_of(v.v[k]);
            }
            if (r < rows && c < columns) *(Pack<Out, 8> *)((Out *)to + p * part + r * to_stride + c) = b;
            *(Pack<Out, 8> *)&tile[p][r0 + h][c8] = b;
        }
    }
    __syncthreads();
    // the columns: eight rows of one at a time
#pragma unroll
    for (int h = 0; h < 64; h += 32) {
        const int c = threadIdx.x % 32 + h, r8 = threadIdx.x / 32 * 8;
        if (column0 + c >= columns || row0 + r8 >= rows) continue;
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            Pack<Out, 8> b;
#pragma unroll
            for (int k = 0; k < 8; k++) b.v[k] = tile[p][r8 + k][c];
            *(Pack<Out, 8> *)((Out *)turned + p * turned_part + (column0 + c) * turned_stride + row0 + r8) = b;
        }
    }
}

// Labels as 32 bits: -1 for ignored examples, -2 for labels that there are not.  With gradients: the factor of every row of P.
__global__ void __launch_bounds__(256) softmax_rows_kernel(const void *labels, int labels_64, long long rows, long long number_of_labels, long long ignored, const float *gradients,
                                                           int gradients_step, float scale, int *out, float *factors, unsigned *largest)
{
    next_may_start();
    wait_for_previous();
    const long long r = (long long)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const long long l = index_at(labels, labels_64, r);
    const int label = l == ignored ? -1 : l < 0 || l >= number_of_labels ? -2 : (int)l;
    out[r] = label;
    if (!factors) return;
    const float f = label == -1 ? 0.f : label == -2 ? __int_as_float(0x7fffffff) : gradients[r * gradients_step] * scale;
    factors[r] = f;
    if (largest && isfinite(f)) atomicMax(largest, __float_as_uint(fabsf(f)));      // of finite magnitudes: the bits have their order
}

// Statistics of two sets of a row's products, joined.
struct JoinSums {
    float top, sum;
    __device__ __forceinline__ static JoinSums none() { return {-INFINITY, 0.f}; }
    __device__ __forceinline__ void join(JoinSums o, float scale)
    {
        const float next = fmaxf(top, o.top);
        if (next == -INFINITY) sum += o.sum;
        else sum = (top == -INFINITY ? sum : sum * expf((top - next) * scale)) + (o.top == -INFINITY ? o.sum : o.sum * expf((o.top - next) * scale));
        top = next;
    }
    __device__ __forceinline__ JoinSums from(int lane_xor) const
    {
        JoinSums o;
        o.top = __shfl_xor_sync(~0u, top, lane_xor), o.sum = __shfl_xor_sync(~0u, sum, lane_xor);
        return o;
    }
    __device__ __forceinline__ static JoinSums read(const float2 *sums, const int *, long long at)
    {
        JoinSums s;
        s.top = sums[at].x, s.sum = sums[at].y;
        return s;
    }
};

struct JoinBest {
    float top, rest;
    int index;
    __device__ __forceinline__ static JoinBest none() { return {-INFINITY, 0.f, 0x7fffffff}; }
    __device__ __forceinline__ void join(JoinBest o, float scale)
    {
        if (o.top == -INFINITY) { rest += o.rest; return; }
        if (top == -INFINITY) { o.rest += rest; *this = o; return; }
        const bool other = o.top > top || (o.top == top && o.index < index);
        const float low = other ? top : o.top, high = other ? o.top : top;
        rest = (other ? o.rest : rest) + (1.f + (other ? rest : o.rest)) * expf((low - high) * scale);
        top = high, index = other ? o.index : index;
    }
    __device__ __forceinline__ JoinBest from(int lane_xor) const
    {
        JoinBest o;
        o.top = __shfl_xor_sync(~0u, top, lane_xor), o.rest = __shfl_xor_sync(~0u, rest, lane_xor), o.index = __shfl_xor_sync(~0u, index, lane_xor);
        return o;
    }
    __device__ __forceinline__ static JoinBest read(const float2 *sums, const int *best, long long at)
    {
        JoinBest s;
        s.top = sums[at].x, s.rest = sums[at].y, s.index = best[at];
        return s;
    }
};

// Joins the parts of kRows rows: a row's parts are read by 1024 / kRows threads, four at a time, joined by warps and then by one warp.  Returns
// the row of the thread and whether it has the result.
template <class J, int kRows>
__device__ __forceinline__ bool join_parts(const float2 *sums, const int *best, long long rows, int parts, float scale, J &mine, long long &row)
{
    constexpr int kEach = 1024 / kRows, kWarps = kEach / 32;          // threads and warps of a row
    __shared__ J shared[kRows][kEach + 1];
    const int x = threadIdx.x % kRows, y = threadIdx.x / kRows;
    const long long from = (long long)blockIdx.x * kRows + x;
    J all = J::none();
    if (from < rows)
        for (int i = y; i < parts; i += 4 * kEach) {
            J part[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k * kEach < parts) part[k] = J::read(sums, best, (long long)(i + k * kEach) * rows + from);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k * kEach < parts) all.join(part[k], scale);
        }
    shared[x][y] = all;
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = warp / kWarps;
    mine = shared[r][warp % kWarps * 32 + lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) mine.join(mine.from(o), scale);
    row = (long long)blockIdx.x * kRows + r;
    if (kWarps == 1) return lane == 0 && row < rows;
    __shared__ J last[32];
    if (lane == 0) last[warp] = mine;
    __syncthreads();
    if (warp) return false;
    mine = last[lane];
#pragma unroll
    for (int o = 1; o < kWarps; o *= 2) mine.join(mine.from(o), scale);
    row = (long long)blockIdx.x * kRows + lane / kWarps;
    return lane % kWarps == 0 && row < rows;
}

template <int kRows>
__global__ void __launch_bounds__(1024) softmax_loss_kernel(const float2 *sums, const float *label_logit, const int *labels, long long rows, int parts, float scale, float *losses,
                                                            float *normalisers)
{
    next_may_start();
    wait_for_previous();
    JoinSums s;
    long long row;
    if (!join_parts<JoinSums, kRows>(sums, nullptr, rows, parts, scale, s, row)) return;
    const float log_sum = logf(s.sum);
    normalisers[row] = fmaf(s.top, scale, log_sum);
    const int label = labels[row];
    losses[row] = label == -1 ? 0.f : label == -2 ? __int_as_float(0x7fffffff) : fmaf(s.top - label_logit[row], scale, log_sum);
}

template <int kRows>
__global__ void __launch_bounds__(1024) softmax_best_kernel(const float2 *sums, const int *best, long long rows, int parts, float scale, long long *labels, float *log_probabilities)
{
    next_may_start();
    wait_for_previous();
    JoinBest s;
    long long row;
    if (!join_parts<JoinBest, kRows>(sums, best, rows, parts, scale, s, row)) return;
    const float log_probability = s.top == -INFINITY ? __int_as_float(0x7fffffff) : -log1pf(s.rest);
    log_probabilities[row] = log_probability;
    labels[row] = log_probability == log_probability ? s.index : -1;
}

// Adds the splits of dw up, in their order, a thread four columns of a row.
template <class T>
__global__ void __launch_bounds__(256) softmax_finish_kernel(const float *partial, long long partial_stride, long long split_size, int splits, long long rows, int columns, const unsigned *out_scale, T *out,
                                                             bool whole)
{
    next_may_start();
    wait_for_previous();
    const float factor = out_scale ? __uint_as_float(*out_scale) * (1.f / 16384.f) : 1.f;
    const int per_row = (columns + 3) / 4;
    const long long all = rows * per_row;
    const bool narrow = all < 1ll << 32;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long r = narrow ? (long long)((unsigned)i / (unsigned)per_row) : i / per_row;
        const int c = (int)(i - r * per_row) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int s = 0; s < splits; s++) {
            const float4 v = *(const float4 *)(partial + s * split_size + r * partial_stride + c);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        Pack<T, 4> q;
        q.v[0] = from_float<T>(sum.x * factor), q.v[1] = from_float<T>(sum.y * factor), q.v[2] = from_float<T>(sum.z * factor), q.v[3] = from_float<T>(sum.w * factor);
        T *to = out + r * columns + c;
        if (whole) *(Pack<T, 4> *)to = q;
        else
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (c + k < columns) to[k] = q.v[k];
    }
}

// Adds the slices of dx up, in their order, and turns it: the product's rows are the columns of features, its columns the examples.  A block has 32 rows
// of a tile and 64 of its columns.
template <class T>
__global__ void __launch_bounds__(256) softmax_turn_kernel(const float *partial, long long partial_stride, long long slice_size, const Product p, const Schedule schedule, const unsigned *out_scale, T *out)
{
    next_may_start();
    wait_for_previous();
    __shared__ float tile[32][65];
    const int across = p.tile_columns / 64, t = blockIdx.x / (8 * across), strip = blockIdx.x / across % 8, part = blockIdx.x % across;
    int m, n;
    p.tile(t, m, n);
    const long long row0 = m * 256ll + strip * 32, column0 = (long long)n * p.tile_columns + part * 64;
    if (row0 >= p.rows || column0 >= p.columns) return;
    const int slices = schedule.slices(p.blocks, t);
    const float factor = out_scale ? __uint_as_float(*out_scale) * (1.f / 16384.f) : 1.f;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        const int r = threadIdx.x / 16 + h, c = threadIdx.x % 16 * 4;
        if (row0 + r < p.rows && column0 + c < p.columns) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            const float *from = partial + (row0 + r) * partial_stride + column0 + c;
#pragma unroll 2
            for (int s = 0; s < slices; s++) {
                const float4 v = *(const float4 *)(from + s * slice_size);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            tile[r][c] = sum.x, tile[r][c + 1] = sum.y, tile[r][c + 2] = sum.z, tile[r][c + 3] = sum.w;
        }
    }
    __syncthreads();
    const int r = threadIdx.x % 32;
    if (row0 + r >= p.rows) return;
    for (int c = threadIdx.x / 32; c < 64 && column0 + c < p.columns; c += 8) out[(column0 + c) * p.rows + row0 + r] = from_float<T>(tile[r][c] * factor);
}

// -------------------------------------------------------------------------------------------------------- host side
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_tiled(EncodeTiled *out)
{
    static std::atomic<EncodeTiled> known;       // the same whichever thread finds it
    EncodeTiled found = known.load();
    if (!found) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult result;
        GTM_CU(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result));
        if (result != cudaDriverEntryPointSuccess || !f) return fail(GTM_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        known.store(found = (EncodeTiled)f);
    }
    *out = found;
    return GTM_OK;
}

// A matrix as the kernels read or write it: rows at 16-byte boundaries, in one part or several.
struct Matrix {
    const void *data;
    int64_t rows, columns, stride, part;         // elements
    int parts;
    int type;
};

int make_map(CUtensorMap *map, const Matrix &a, unsigned box_columns, unsigned box_rows)
{
    EncodeTiled encode;
    GTM_TRY(encode_tiled(&encode));
    const cuuint64_t size = type_bytes(a.type);
    const cuuint64_t sizes[3] = {(cuuint64_t)a.columns, (cuuint64_t)a.rows, (cuuint64_t)a.parts};
    const cuuint64_t strides[2] = {(cuuint64_t)a.stride * size, (cuuint64_t)(a.parts > 1 ? a.part : a.stride) * size};      // of one part: any
    const cuuint32_t box[3] = {box_columns, box_rows, 1}, steps[3] = {1, 1, 1};
    const CUtensorMapDataType kind = a.type == GTM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : a.type == GTM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, kind, 3, (void *)a.data, sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GTM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %lld x %lld elements, stride %lld", (int)r, (long long)a.rows, (long long)a.columns, (long long)a.stride);
    return GTM_OK;
}

__device__ unsigned softmax_error;               // counts waits that ran out

constexpr unsigned long long kWait = 10000000000ull, kShortWait = 50000000ull;      // nanoseconds
thread_local int lost_launches;                  // of the calling thread that are to come: their waits run out

int set_operands(Maps &maps, Product &p, int which, const Matrix &a, const Matrix &b, const Matrix *out)
{
    GTM_TRY(make_map(&maps.a[which], a, 64, p.a_rows ? 64 : 128));
    GTM_TRY(make_map(&maps.b[which], b, 64, p.tile_columns / 2));
    if (out) GTM_TRY(make_map(&maps.out[which], *out, out->type == GTM_F32 ? 32 : 64, 32));
    p.what = product(a.type == GTM_F16 ? 0 : 1, p.tile_columns, p.a_rows);
    return GTM_OK;
}

template <int kMode>
int launch_product(const Maps &maps, Launch &l, cudaStream_t stream)
{
    // what does not change on a device is asked for once
    static std::atomic<void *> errors[64];
    int device = 0;
    GTM_CU(cudaGetDevice(&device));
    void *error = device < 64 ? errors[device].load() : nullptr;
    if (!error) {
        GTM_CU(cudaGetSymbolAddress(&error, softmax_error));
        GTM_CU(cudaFuncSetAttribute(softmax_product_kernel<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_of(kMode)));
        if (kMode != kOut) {
            // built otherwise, its epilogue would wait for registers for good
            cudaFuncAttributes built;
            GTM_CU(cudaFuncGetAttributes(&built, softmax_product_kernel<kMode>));
            if (built.numRegs < kLaunchedRegisters) return fail(GTM_ERR_CUDA, "the product kernel is built for %d registers a thread instead of %d", built.numRegs, kLaunchedRegisters);
        }
        if (device < 64) errors[device].store(error);
    }
    l.error = (unsigned *)error;
    l.limit = kWait, l.lost = 0;
    if (lost_launches > 0) lost_launches--, l.limit = kShortWait, l.lost = 1;
    const unsigned pairs = (unsigned)(l.schedule.units ? l.schedule.pairs : std::min(l.schedule.items, l.schedule.pairs));
    return launch_early(softmax_product_kernel<kMode>, dim3(2 * pairs), dim3(kThreads), shared_of(kMode), stream, maps, l);
}

// Tiles of 128 columns take nearly as long as those of 256 (0.42 us a block of the sum's index against 0.46: what both wait for is operand A), so
// they are for results that have no more columns, and for those of which all tiles of 128 are at work at once.
int tile_columns(int64_t rows, int64_t columns)
{
    return columns <= 128 || (rows + 255) / 256 * ((columns + 127) / 128) <= kPairs ? 128 : 256;
}

Product product_of(int64_t rows, int64_t columns, int64_t depth, int products, int tile = 0)
{
    Product p = {};
    p.rows = rows, p.columns = columns, p.products = products;
    p.tile_columns = tile ? tile : tile_columns(rows, columns);
    p.m_tiles = (int)((rows + 255) / 256), p.n_tiles = (int)((columns + p.tile_columns - 1) / p.tile_columns);
    p.depth_blocks = (int)((depth + kDepth - 1) / kDepth);
    p.blocks = p.per_split = p.depth_blocks * products;
    p.chunk = p.depth_blocks;
    return p;
}

// Blocks of the index whose products follow each other in tensor memory, for logits.  What the tensor cores cut off a sum grows with the square of its steps, so there
// are up to five blocks (320 elements, 20 steps), two for 32-bit inputs, and two sums from three blocks on; losses of 16-bit inputs are then 0.5 to 1.2 times as far from
// 64 bits as those of plain 32-bit products, from 130 to 2,048 columns.  Statistics of 8,192 x 1,024 bf16 and 65,536 labels take 833 us so (four sums), 814 in three, 787 in two
// (errors 1.4 times larger), 900 in six: the epilogue reads tensor memory while products write to it.
int logits_chunk(const Product &p)
{
    const int most = p.products == 1 ? 5 : 2, chunks = std::max((p.depth_blocks + most - 1) / most, p.depth_blocks > 2 ? 2 : 1);
    return (p.depth_blocks + chunks - 1) / chunks;
}

// One product alone, its tiles in turn.
Schedule in_turn(const Product &p) { return {p.tiles() * p.splits(), kPairs, 0, kPairs, 0, 0}; }

// Two products; weights are blocks, an epilogue being worth about six of them.  No pair has less than eight blocks of the second product
// (or one pair has them all): slices cost, and a pair without work would leave one unwritten.
constexpr int kLeastShare = 8;
Schedule together(const Product &first, const Product &second)
{
    Schedule s = {first.tiles() * first.splits(), kPairs, 0, kPairs, (long long)second.tiles() * second.blocks, 0};
    const double item = first.per_split + 6.0, unit = 1.0;
    s.longer = s.items % kPairs;
    if (s.longer) {
        const double each = (s.units * unit - (kPairs - s.longer) * item) / kPairs;     // what is left for a longer pair
        if (each > (kLeastShare + 1) * unit) s.units_of_longer = std::min(s.units, (long long)(each * s.longer / unit));
    }
    s.others = (int)std::max<long long>(1, std::min<long long>(kPairs - s.longer, (s.units - s.units_of_longer) / kLeastShare));
    return s;
}

int most_slices(const Schedule &s, const Product &p)
{
    if (p.tiles() > 64) {
        // a bound: by the smallest share that a pair has
        long long least = (s.units - s.units_of_longer) / s.others;
        if (least == 0 || (s.units_of_longer && s.units_of_longer / s.longer < least)) least = s.units_of_longer / s.longer;
        return (int)std::min<long long>(kPairs, p.blocks / least + 2);
    }
    int most = 1;
    for (int t = 0; t < p.tiles(); t++) most = std::max(most, s.slices(p.blocks, t));
    return most;
}

// What a call reads, and where its workspace's parts are.
struct Call {
    int type, products, parts;
    int64_t examples, labels, columns;
    const void *x, *w;
    int64_t x_stride, w_stride;
    bool lay_out_x, lay_out_w, gradient, predict;
    int64_t x_ld, w_ld;
    // forward
    bool few, few_whole;
    int64_t piece_rows;
    int stat_parts;
    // gradient
    int64_t piece_labels, prob_ld, sums_ld, turned_ld;
    Product dx, dw;
    Schedule schedule;
    int dx_slices;
    bool dw_direct;
    uint64_t at_x, at_turned, at_w, at_rows, at_factors, at_largest, at_sums, at_best, at_logit, at_prob, at_dx, at_dw, total;
};

bool direct(int type, const void *p, int64_t rows, int64_t stride, int64_t columns)
{
    return type != GTM_F32 && (uintptr_t)p % 16 == 0 && (rows == 1 || (stride * 2 % 16 == 0 && stride >= columns));
}

int64_t clamp64(int64_t v, int64_t low, int64_t high) { return v < low ? low : v > high ? high : v; }

// A piece of the labels: P of it within kPieceBytes, and as few rounds of tiles over all pieces as that allows.
int64_t piece_of(int64_t examples, int64_t labels, int parts)
{
    const int64_t m_tiles = (examples + 255) / 256, all = (labels + 255) / 256;
    const int64_t most = std::min(all, clamp64(kPieceBytes / (examples * 2 * parts) / 256, 1, 4096));
    if (most == all) return labels;
    int64_t best = most, least = -1;
    for (int64_t tiles = most; tiles >= std::max<int64_t>(1, most / 2); tiles--) {
        const int64_t rounds = (all + tiles - 1) / tiles * ((m_tiles * tiles + kPairs - 1) / kPairs);
        if (least < 0 || rounds < least) least = rounds, best = tiles;
    }
    return best * 256;
}

constexpr int few_blocks(size_t element, int examples) { return 148 * (few_rows(element, examples) == 4 ? 4 : 8); }
constexpr size_t kFewShared = 96 << 10;

void lay_out_workspace(Call &c)
{
    c.products = c.type == GTM_F32 ? kPartProducts : 1;
    c.parts = c.type == GTM_F32 ? 3 : 1;
    const int64_t size = (int64_t)type_bytes(c.type);
    // as many examples as are multiplied by the plain units about as fast as memory delivers the weights: 8 in 32 bits (and no parts to lay out), 2 in 16
    const int64_t padded = (int64_t)round_up(c.columns, 256);
    c.few = c.predict && c.examples <= (c.type == GTM_F32 ? 8 : 2) && (c.examples <= 4 ? 4 : 8) * padded * 4 <= (int64_t)kFewShared;
    c.few_whole = aligned(c.w, c.w_stride * size, 16) && c.columns * size % 16 == 0;
    // the gradient's x is laid out anew in any case: examples that are ignored may hold anything
    c.lay_out_x = !c.few && (c.gradient || !direct(c.type, c.x, c.examples, c.x_stride, c.columns));
    c.lay_out_w = !c.few && !direct(c.type, c.w, c.labels, c.w_stride, c.columns);
    const int64_t ld = (int64_t)round_up(c.columns, 8);
    c.x_ld = c.lay_out_x || c.examples == 1 ? ld : c.x_stride;
    c.w_ld = c.lay_out_w || c.labels == 1 ? ld : c.w_stride;
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) { const uint64_t here = at; at += round_up(bytes, 256); return here; };
    c.at_x = take(c.lay_out_x ? (uint64_t)c.parts * c.examples * ld * 2 : 0);
    c.at_w = take(c.lay_out_w ? (uint64_t)c.parts * c.labels * ld * 2 : 0);
    c.at_rows = take(c.examples * 4);
    if (!c.gradient) {
        const int tile = tile_columns(c.examples, c.labels);
        c.stat_parts = c.few ? few_blocks(size, (int)c.examples) : (int)((c.labels + tile - 1) / tile) * 2;
        c.piece_rows = std::min<int64_t>(c.examples, clamp64(kStatBytes / (c.stat_parts * 8) / 256 * 256, 256, (int64_t)1 << 30));
        c.at_sums = take((uint64_t)c.stat_parts * c.piece_rows * 8);
        c.at_best = take((uint64_t)c.stat_parts * c.piece_rows * 4);
        c.at_logit = take(c.piece_rows * 4);
    } else {
        c.at_factors = take(c.examples * 4);
        c.at_largest = take(4);
        c.piece_labels = piece_of(c.examples, c.labels, c.parts);
        // a piece's sums of dx are cut as well, by pairs of SMs that share a tile
        const int64_t dx_tiles = ((c.columns + 255) / 256) * ((c.examples + 255) / 256);
        if (c.products == 1) c.piece_labels = std::min(c.piece_labels, kLongestSum * kDepth * std::max<int64_t>(1, kPairs / dx_tiles));
        c.prob_ld = (int64_t)round_up(c.piece_labels, 64);
        c.sums_ld = (int64_t)round_up(c.columns, 4);
        c.turned_ld = (int64_t)round_up(c.examples, 8);
        c.at_turned = take((uint64_t)c.parts * c.columns * c.turned_ld * 2);
        c.at_prob = take((uint64_t)c.parts * c.examples * c.prob_ld * 2);
        c.dx = product_of(c.columns, c.examples, c.piece_labels, c.products, c.examples <= 128 ? 128 : 256);      // turned: its operand B is P
        c.dw = product_of(c.piece_labels, c.columns, c.examples, c.products);
        if (c.products > 1) c.dx.chunk = c.dw.chunk = 8;
        // dw's tiles are cut where they are less than half of the pairs of SMs, into eight blocks or more, and where sums would be too long
        const int splits = std::max(std::max(1, std::min(kPairs / c.dw.tiles(), c.dw.blocks / 8)), c.products == 1 ? (c.dw.blocks + kLongestSum - 1) / kLongestSum : 1);
        c.dw.per_split = (c.dw.blocks + splits - 1) / splits;
        c.schedule = together(c.dw, c.dx);
        c.dx_slices = most_slices(c.schedule, c.dx);
        c.dw_direct = c.dw.splits() == 1 && c.columns * size % 16 == 0;
        c.at_dx = take((uint64_t)c.dx_slices * c.columns * c.turned_ld * 4);
        c.at_dw = take(c.dw_direct ? 0 : (uint64_t)c.dw.splits() * c.piece_labels * c.sums_ld * 4);
    }
    c.total = at;
}

int check_call(const char *what, const Call &c, float scale)
{
    if (!type_bytes(c.type)) return fail(GTM_ERR_ARG, "%s: element type %d is none of GTM_F32, GTM_BF16, GTM_F16", what, c.type);
    if (c.examples < 0 || c.examples >= kMostRows / 256) return fail(GTM_ERR_ARG, "%s: %lld examples (below 2^23)", what, (long long)c.examples);
    if (c.labels < 1 || c.labels >= kMostRows / 4) return fail(GTM_ERR_ARG, "%s: %lld labels (1 to 2^29 - 1)", what, (long long)c.labels);
    if (c.columns < 1 || c.columns > (1 << 20)) return fail(GTM_ERR_ARG, "%s: %lld columns (1 to 2^20)", what, (long long)c.columns);
    if (c.x_stride < 0 || c.w_stride < 0) return fail(GTM_ERR_ARG, "%s: negative row stride", what);
    if ((uintptr_t)c.x % type_bytes(c.type) || (uintptr_t)c.w % type_bytes(c.type)) return fail(GTM_ERR_ARG, "%s: an array does not start at a boundary of its elements", what);
    if (!(scale > 0.f) || scale > 3.4e38f) return fail(GTM_ERR_ARG, "%s: scale %g is not above zero and finite", what, (double)scale);
    return GTM_OK;
}

int check_workspace(const char *what, const void *workspace, uint64_t bytes, uint64_t need)
{
    if (bytes < need || !workspace || (uintptr_t)workspace % 256)
        return fail(GTM_ERR_ARG, "%s: workspace of %llu bytes, %llu needed (256-byte aligned)", what, (unsigned long long)bytes, (unsigned long long)need);
    return GTM_OK;
}

template <class T>
int lay_out(const void *from, int64_t stride, int64_t rows, int64_t columns, const int *labels, void *to, int64_t ld, cudaStream_t stream)
{
    const int64_t blocks = std::min<int64_t>((rows * ((columns + 7) / 8) + 255) / 256, 148 * 16);
    const bool whole = aligned(from, stride * sizeof(T), 16) && columns % 8 == 0;
    return launch_early(whole ? softmax_lay_out_kernel<T, true> : softmax_lay_out_kernel<T, false>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T *)from, (long long)stride, (long long)rows, (int)columns,
                        labels, (__nv_bfloat16 *)to, (long long)ld, (long long)(rows * ld));
}

// A matrix as the kernels read it, laid out in the workspace where it is not so already.
int operand_of(Matrix *out, int type, const void *data, int64_t stride, int64_t rows, int64_t columns, bool copy, const int *labels, void *to, int64_t ld, cudaStream_t stream)
{
    if (copy) {
        GTM_TRY(type == GTM_F32    ? lay_out<float>(data, stride, rows, columns, labels, to, ld, stream)
                : type == GTM_BF16 ? lay_out<__nv_bfloat16>(data, stride, rows, columns, labels, to, ld, stream)
                                   : lay_out<__half>(data, stride, rows, columns, labels, to, ld, stream));
        data = to;
    }
    *out = {data, rows, columns, ld, rows * ld, type == GTM_F32 ? 3 : 1, type == GTM_F16 ? GTM_F16 : GTM_BF16};
    return GTM_OK;
}

template <class T>
int lay_out_both(const Call &c, const int *labels, char *w, cudaStream_t stream)
{
    const dim3 grid((unsigned)((c.examples + 63) / 64), (unsigned)((c.columns + 63) / 64));
    const bool whole = aligned(c.x, c.x_stride * sizeof(T), 16) && c.columns % 8 == 0;
    return launch_early(softmax_lay_out_both_kernel<T>, grid, dim3(256), 0, stream, (const T *)c.x, (long long)c.x_stride, (long long)c.examples, (int)c.columns, labels, (__nv_bfloat16 *)(w + c.at_x),
                        (long long)c.x_ld, (long long)(c.examples * c.x_ld), (__nv_bfloat16 *)(w + c.at_turned), (long long)c.turned_ld, (long long)(c.columns * c.turned_ld), whole);
}

template <class T>
int finish_dw(const Call &c, const float *dw, int64_t rows, const unsigned *out_scale, void *out, cudaStream_t stream)
{
    const unsigned blocks = (unsigned)std::min<int64_t>((rows * ((c.columns + 3) / 4) + 255) / 256, 148 * 16);
    return launch_early(softmax_finish_kernel<T>, dim3(blocks), dim3(256), 0, stream, dw, (long long)c.sums_ld, (long long)(c.piece_labels * c.sums_ld), c.dw.splits(), (long long)rows, (int)c.columns, out_scale,
                        (T *)out, c.columns % 4 == 0);
}

template <class T>
int finish_dx(const Call &c, const float *dx, const unsigned *out_scale, void *out, cudaStream_t stream)
{
    return launch_early(softmax_turn_kernel<T>, dim3((unsigned)(c.dx.tiles() * 8 * (c.dx.tile_columns / 64))), dim3(256), 0, stream, dx, (long long)c.turned_ld, (long long)(c.columns * c.turned_ld), c.dx, c.schedule,
                        out_scale, (T *)out);
}

template <class T, int kExamples, bool kWhole>
int launch_few(const FewArgs &a, int blocks, cudaStream_t stream)
{
    const size_t shared = kExamples * round_up(a.columns, 256) * 4;
    GTM_CU(cudaFuncSetAttribute(softmax_few_kernel<T, kExamples, kWhole>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewShared));
    return launch_early(softmax_few_kernel<T, kExamples, kWhole>, dim3(blocks), dim3(kFewThreads), shared, stream, a);
}

template <class T>
int launch_few(const FewArgs &a, bool whole, int blocks, cudaStream_t stream)
{
    if (a.examples == 1) return whole ? launch_few<T, 1, true>(a, blocks, stream) : launch_few<T, 1, false>(a, blocks, stream);
    if (a.examples == 2) return whole ? launch_few<T, 2, true>(a, blocks, stream) : launch_few<T, 2, false>(a, blocks, stream);
    if constexpr (sizeof(T) == 4) {
        if (a.examples <= 4) return whole ? launch_few<T, 4, true>(a, blocks, stream) : launch_few<T, 4, false>(a, blocks, stream);
        return whole ? launch_few<T, 8, true>(a, blocks, stream) : launch_few<T, 8, false>(a, blocks, stream);
    }
    return fail(GTM_ERR_ARG, "more examples than are few");
}

// Rows per block of the kernels that join parts: as few as there are.
template <class Run>
int by_rows(int64_t rows, Run run)
{
    if (rows <= 8) return run(std::integral_constant<int, 1>(), dim3((unsigned)rows));
    if (rows <= 148 * 8) return run(std::integral_constant<int, 8>(), dim3((unsigned)((rows + 7) / 8)));
    return run(std::integral_constant<int, 32>(), dim3((unsigned)((rows + 31) / 32)));
}

// Loss (labels given) or most probable label.
int forward(Call &c, const void *labels, int labels_64, int64_t ignored, float scale, float *losses, float *normalisers, int64_t *best, float *log_probabilities, char *w, cudaStream_t stream)
{
    int *rows = labels ? (int *)(w + c.at_rows) : nullptr;
    if (labels) {
        GTM_TRY(launch_early(softmax_rows_kernel, dim3((unsigned)((c.examples + 255) / 256)), dim3(256), 0, stream, labels, labels_64, (long long)c.examples, (long long)c.labels, (long long)ignored,
                             nullptr, 0, scale, rows, nullptr, nullptr));
    }
    float2 *sums = (float2 *)(w + c.at_sums);
    int *indices = (int *)(w + c.at_best);
    float *label_logit = (float *)(w + c.at_logit);
    const auto join = [&](int64_t first, int64_t n, int parts, float scale) {
        return by_rows(n, [&](auto each, dim3 blocks) -> int {
            constexpr int kRows = decltype(each)::value;
            if (labels)
                return launch_early(softmax_loss_kernel<kRows>, blocks, dim3(1024), 0, stream, sums, label_logit, rows + first, (long long)n, parts, scale, losses + first, normalisers + first);
            return launch_early(softmax_best_kernel<kRows>, blocks, dim3(1024), 0, stream, sums, indices, (long long)n, parts, scale, (long long *)best + first, log_probabilities + first);
        });
    };
    if (c.few) {
        const FewArgs a = {c.x, c.w, c.x_stride, c.w_stride, (int)c.examples, (int)c.labels, (int)c.columns, scale, sums, indices};
        const size_t size = type_bytes(c.type);
        const int64_t turn = few_rows(size, (int)c.examples) * (kFewThreads / 32);
        const int blocks = (int)std::min<int64_t>(few_blocks(size, (int)c.examples), (c.labels + turn - 1) / turn);
        GTM_TRY(c.type == GTM_F32    ? launch_few<float>(a, c.few_whole, blocks, stream)
                : c.type == GTM_BF16 ? launch_few<__nv_bfloat16>(a, c.few_whole, blocks, stream)
                                     : launch_few<__half>(a, c.few_whole, blocks, stream));
        return join(0, c.examples, blocks, scale);
    }
    Matrix x, weights;
    GTM_TRY(operand_of(&x, c.type, c.x, c.x_stride, c.examples, c.columns, c.lay_out_x, nullptr, w + c.at_x, c.x_ld, stream));
    GTM_TRY(operand_of(&weights, c.type, c.w, c.w_stride, c.labels, c.columns, c.lay_out_w, nullptr, w + c.at_w, c.w_ld, stream));
    for (int64_t r = 0; r < c.examples; r += c.piece_rows) {
        const int64_t n = std::min(c.piece_rows, c.examples - r);
        Matrix piece = x;
        piece.data = (const char *)x.data + r * x.stride * 2;
        piece.rows = n;
        Launch l = {};
        Maps maps = {};
        Product &p = l.p[0] = product_of(n, c.labels, c.columns, c.products, tile_columns(c.examples, c.labels));      // as the workspace has it
        p.m_fast = 1, p.chunk = logits_chunk(p);
        l.schedule = in_turn(p);
        l.scale = scale, l.sums = sums, l.best = indices, l.label_logit = label_logit, l.labels = labels ? rows + r : nullptr;
        GTM_TRY(set_operands(maps, p, 0, piece, weights, nullptr));
        if (labels) GTM_TRY(launch_product<kSums>(maps, l, stream));
        else GTM_TRY(launch_product<kBest>(maps, l, stream));
        GTM_TRY(join(r, n, p.n_tiles * 2, scale));
    }
    return GTM_OK;
}

}  // namespace
}  // namespace gtm_readout

using namespace gtm_readout;

enum { kLossCall, kGradientCall, kPredictCall };

static Call call_of(int type, int64_t examples, int64_t labels, int64_t columns, const void *x, int64_t x_stride, const void *w, int64_t w_stride, int what)
{
    Call c = {};
    c.type = type, c.examples = examples, c.labels = labels, c.columns = columns, c.x = x, c.w = w, c.x_stride = x_stride, c.w_stride = w_stride, c.gradient = what == kGradientCall, c.predict = what == kPredictCall;
    return c;
}

extern "C" int gtm_softmax_workspace(int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t labels, int64_t weights_stride,
                                     int64_t columns, int what, uint64_t *bytes_out)
{
    if (!bytes_out) return fail(GTM_ERR_ARG, "gtm_softmax_workspace: null output");
    if (what < kLossCall || what > kPredictCall) return fail(GTM_ERR_ARG, "gtm_softmax_workspace: call %d (0: loss, 1: gradient, 2: prediction)", what);
    Call c = call_of(type, examples, labels, columns, features, features_stride, weights, weights_stride, what);
    GTM_TRY(check_call("gtm_softmax_workspace", c, 1.f));
    *bytes_out = 0;
    if (examples == 0) return GTM_OK;
    if (few_labels(examples, labels, columns)) {
        *bytes_out = few_labels_workspace(examples, labels, columns, c.gradient);
        return GTM_OK;
    }
    lay_out_workspace(c);
    *bytes_out = c.total;
    return GTM_OK;
}

extern "C" int gtm_softmax_loss(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t number_of_labels,
                                int64_t weights_stride, int64_t columns, const void *labels, int labels_64, int64_t ignore_label, float scale, float *losses, float *normalisers,
                                void *workspace, uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, kLossCall);
    GTM_TRY(check_call("gtm_softmax_loss", c, scale));
    if (examples == 0) return GTM_OK;
    if (!features || !weights || !labels || !losses || !normalisers) return fail(GTM_ERR_ARG, "gtm_softmax_loss: null array");
    const bool few_ones = few_labels(examples, number_of_labels, columns);
    if (!few_ones) {
        lay_out_workspace(c);
        GTM_TRY(check_workspace("gtm_softmax_loss", workspace, workspace_bytes, c.total));
    }
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    if (few_ones) {
        const FewLabels few = {type, examples, number_of_labels, columns, features, weights, features_stride, weights_stride, labels, labels_64, ignore_label, scale};
        return few_labels_loss(few, losses, normalisers, (cudaStream_t)cuda_stream);
    }
    return forward(c, labels, labels_64, ignore_label, scale, losses, normalisers, nullptr, nullptr, (char *)workspace, (cudaStream_t)cuda_stream);
}

extern "C" int gtm_softmax_predict(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t number_of_labels,
                                   int64_t weights_stride, int64_t columns, float scale, int64_t *labels_out, float *log_probabilities_out, void *workspace, uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, kPredictCall);
    GTM_TRY(check_call("gtm_softmax_predict", c, scale));
    if (examples == 0) return GTM_OK;
    if (!features || !weights || !labels_out || !log_probabilities_out) return fail(GTM_ERR_ARG, "gtm_softmax_predict: null array");
    const bool few_ones = few_labels(examples, number_of_labels, columns);
    if (!few_ones) {
        lay_out_workspace(c);
        GTM_TRY(check_workspace("gtm_softmax_predict", workspace, workspace_bytes, c.total));
    }
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    if (few_ones) {
        const FewLabels few = {type, examples, number_of_labels, columns, features, weights, features_stride, weights_stride, nullptr, 0, 0, scale};
        return few_labels_predict(few, labels_out, log_probabilities_out, (cudaStream_t)cuda_stream);
    }
    return forward(c, nullptr, 0, 0, scale, nullptr, nullptr, labels_out, log_probabilities_out, (char *)workspace, (cudaStream_t)cuda_stream);
}

extern "C" int gtm_softmax_loss_gradient(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights,
                                         int64_t number_of_labels, int64_t weights_stride, int64_t columns, const void *labels, int labels_64, int64_t ignore_label, float scale,
                                         const float *normalisers, const float *gradients, int64_t gradients_step, void *features_gradient, void *weights_gradient, void *workspace,
                                         uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, kGradientCall);
    GTM_TRY(check_call("gtm_softmax_loss_gradient", c, scale));
    if (!weights_gradient || (uintptr_t)weights_gradient % 16 || (uintptr_t)features_gradient % 16)
        return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: a result is null or does not start at a 16-byte boundary");
    if (gradients_step != 0 && gradients_step != 1) return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: step %lld of the gradients (0 or 1)", (long long)gradients_step);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    if (examples == 0) {
        GTM_CU(cudaMemsetAsync(weights_gradient, 0, (size_t)number_of_labels * columns * type_bytes(type), stream));
        return GTM_OK;
    }
    if (!features || !weights || !labels || !normalisers || !gradients || !features_gradient) return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: null array");
    if (few_labels(examples, number_of_labels, columns)) {
        GTM_TRY(check_workspace("gtm_softmax_loss_gradient", workspace, workspace_bytes, few_labels_workspace(examples, number_of_labels, columns, true)));
        const FewLabels few = {type, examples, number_of_labels, columns, features, weights, features_stride, weights_stride, labels, labels_64, ignore_label, scale};
        return few_labels_gradient(few, normalisers, gradients, gradients_step, features_gradient, weights_gradient, workspace, stream);
    }
    lay_out_workspace(c);
    GTM_TRY(check_workspace("gtm_softmax_loss_gradient", workspace, workspace_bytes, c.total));
    char *w = (char *)workspace;
    int *rows = (int *)(w + c.at_rows);
    float *factors = (float *)(w + c.at_factors);
    unsigned *largest = type == GTM_F16 ? (unsigned *)(w + c.at_largest) : nullptr;
    if (largest) GTM_CU(cudaMemsetAsync(largest, 0, 4, stream));
    GTM_TRY(launch_early(softmax_rows_kernel, dim3((unsigned)((examples + 255) / 256)), dim3(256), 0, stream, labels, labels_64, (long long)examples, (long long)number_of_labels, (long long)ignore_label,
                         gradients, (int)gradients_step, scale, rows, factors, largest));
    GTM_TRY(type == GTM_F32 ? lay_out_both<float>(c, rows, w, stream) : type == GTM_BF16 ? lay_out_both<__nv_bfloat16>(c, rows, w, stream) : lay_out_both<__half>(c, rows, w, stream));
    const int held = type == GTM_F16 ? GTM_F16 : GTM_BF16;
    const Matrix x = {w + c.at_x, examples, columns, c.x_ld, examples * c.x_ld, c.parts, held}, turned = {w + c.at_turned, columns, examples, c.turned_ld, columns * c.turned_ld, c.parts, held};
    Matrix wm;
    GTM_TRY(operand_of(&wm, type, weights, weights_stride, number_of_labels, columns, c.lay_out_w, nullptr, w + c.at_w, c.w_ld, stream));
    float *dx = (float *)(w + c.at_dx), *dw = (float *)(w + c.at_dw);
    const int64_t size = (int64_t)type_bytes(type), x_bytes = examples * columns * 2 * c.parts;
    for (int64_t v = 0; v < number_of_labels; v += c.piece_labels) {
        const int64_t n = std::min(c.piece_labels, number_of_labels - v);
        const Matrix prob = {w + c.at_prob, examples, n, c.prob_ld, examples * c.prob_ld, c.parts, held};
        Matrix piece = wm;                        // rows behind the piece read as zeros
        piece.rows = v + n;
        // P of the piece
        {
            Launch l = {};
            Maps maps = {};
            Product &p = l.p[0] = product_of(examples, n, columns, c.products);
            // x stays in L2 while the labels pass, or the piece's labels while the examples do
            p.m_fast = x_bytes <= 64 << 20 || x_bytes <= n * columns * 2 * c.parts, p.b_row = (int)v, p.type = type, p.chunk = logits_chunk(p);
            l.schedule = in_turn(p);
            l.scale = scale, l.labels = rows, l.first_label = (int)v, l.normalisers = normalisers, l.factors = factors, l.largest = largest;
            GTM_TRY(set_operands(maps, p, 0, x, piece, &prob));
            GTM_TRY(launch_product<kProb>(maps, l, stream));
        }
        // dw of the piece, P turned times x, and its share of dx turned, w turned times P.  A last piece that is smaller has the work of a whole one, zeros
        // among it, so that the slices of dx are the same
        Launch l = {};
        Maps maps = {};
        l.schedule = c.schedule;
        Product &pw = l.p[0] = c.dw, &px = l.p[1] = c.dx;
        char *to = (char *)weights_gradient + v * columns * size;
        pw.a_rows = 1, pw.rows = n, pw.type = c.dw_direct ? type : GTM_F32, pw.out_scale = c.dw_direct ? largest : nullptr;
        px.a_rows = 1, px.a_first = (int)v, px.type = GTM_F32, px.add = v > 0;
        const Matrix dw_out = c.dw_direct ? Matrix{to, n, columns, columns, 0, 1, type} : Matrix{dw, n, columns, c.sums_ld, c.piece_labels * c.sums_ld, pw.splits(), GTM_F32};
        const Matrix dx_out = {dx, columns, examples, c.turned_ld, columns * c.turned_ld, c.dx_slices, GTM_F32};
        GTM_TRY(set_operands(maps, pw, 0, prob, turned, &dw_out));
        GTM_TRY(set_operands(maps, px, 1, piece, prob, &dx_out));
        GTM_TRY(launch_product<kOut>(maps, l, stream));
        if (!c.dw_direct)
            GTM_TRY(type == GTM_F32 ? finish_dw<float>(c, dw, n, largest, to, stream) : type == GTM_BF16 ? finish_dw<__nv_bfloat16>(c, dw, n, largest, to, stream) : finish_dw<__half>(c, dw, n, largest, to, stream));
    }
    return type == GTM_F32    ? finish_dx<float>(c, dx, largest, features_gradient, stream)
           : type == GTM_BF16 ? finish_dx<__nv_bfloat16>(c, dx, largest, features_gradient, stream)
                              : finish_dx<__half>(c, dx, largest, features_gradient, stream);
}

extern "C" int gtm_softmax_failed(int device, int *failed_out)
{
    static thread_local unsigned known[64];      // counts that the thread was told of: no question hides a failure from another thread
    if (!failed_out) return fail(GTM_ERR_ARG, "gtm_softmax_failed: null output");
    if (device < 0 || device >= 64) return fail(GTM_ERR_ARG, "gtm_softmax_failed: device %d (0 to 63)", device);
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    unsigned count = 0;
    GTM_CU(cudaDeviceSynchronize());
    GTM_CU(cudaMemcpyFromSymbol(&count, softmax_error, sizeof count));
    *failed_out = count != known[device];
    known[device] = count;
    return GTM_OK;
}

extern "C" int gtm_debug_softmax_lose(int launches)
{
    if (launches < 0) return fail(GTM_ERR_ARG, "gtm_debug_softmax_lose: %d launches", launches);
    lost_launches = launches;
    return GTM_OK;
}
