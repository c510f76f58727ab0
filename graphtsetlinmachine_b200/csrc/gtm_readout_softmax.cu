// Softmax cross entropy over many labels, its gradient, and the most probable label.
//
//   l[n, v] = scale * x[n] . w[v]        lse[n] = log sum_v exp l[n, v]        loss[n] = lse[n] - l[n, label[n]]
//   P = (softmax(l) - onehot(label)) * gradient[n] * scale        dx = P w        dw = P^T x
//
// The logits are never kept.  Forward, a tile of them stays in tensor memory and leaves the largest value and the sum of exponentials of
// every row, which a second kernel joins.  Backward, the labels are taken in pieces: a piece's logits are computed again, P of
// the piece goes to the workspace in the operands' 16-bit type, and two products use it.  All products are one kernel on
// tcgen05 over pairs of thread blocks: tiles of 256 x 256 (or 128), operands by TMA through a ring in shared memory, sums in tensor
// memory, two tiles deep, so that a tile's epilogue runs under the next tile's products.
//
// 16-bit inputs are multiplied as they are, with sums in 32 bits.  32-bit inputs are split into three bf16 parts (24 bits of fraction),
// and the six products of parts that reach 2^-24 are added, the smallest first.  P is rounded to the operands' type, to as many bits as
// dx and dw are; fp16 has too small a range for that, so P is scaled by 2^14 over the largest |gradient * scale| there.
#include "gtm_readout.cuh"
#include "gtm_readout_mma.cuh"

#include <algorithm>

namespace gtm_readout {
namespace {

constexpr int kStages = 6, kDepth = 64;                    // ring, and elements of a sum's index per stage
constexpr int kHalfBytes = 128 * kDepth * 2;               // an operand's share of a stage in one thread block
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kThreads = 384, kEpilogue = 8;               // warps 0: copies, 1: products, 2: tensor memory; 4..11: epilogue
constexpr int kPairs = 74;                                 // pairs of SMs
constexpr size_t kShared = 1024 + kStages * kStageBytes;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kPieceBytes = 128 << 20;                 // of P in the workspace at a time
constexpr int64_t kStatBytes = 64 << 20;                   // of partial sums of exponentials at a time

enum Epilogue { kSums = 0, kBest = 1, kProb = 2, kOut = 3 };

// Parts of a 32-bit operand that are multiplied, the smallest products first: pairs (a, b) of two bits each.
constexpr int kPartProducts = 6;
__device__ __forceinline__ void parts_of(int products, int i, int &a, int &b)
{
    constexpr unsigned as = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10, bs = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;
    a = products == 1 ? 0 : as >> (2 * i) & 3;
    b = products == 1 ? 0 : bs >> (2 * i) & 3;
}

struct Problem {
    long long rows, columns;                    // of the result
    int m_tiles, n_tiles, splits, tile_columns; // 256 or 128 columns of a tile
    int m_fast;                                 // tiles of one column block follow each other
    int depth_blocks, products, per_split;      // blocks of kDepth of the sum's index; blocks (times products) of a split
    int a_rows, b_rows;                         // operands whose rows, not the sum's index, lie next to each other
    int a_first, b_first;                       // offset of the sum's index in the operand's tensor (a row of W)
    int b_row;                                  // offset of the result's columns in operand B (a row of W)
    unsigned what;                              // instruction descriptor
    int *error;
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
    const unsigned *largest;                    // bits of the largest |factor|, null: factors as they are
    void *prob;
    long long prob_stride, prob_part;           // elements
    // kProb, kOut
    int type;                                   // of the result
    // kOut
    void *out;
    long long out_stride;
    float *partial;                             // [split][rows][columns], instead of out
    int add;                                    // to what partial holds
    const unsigned *out_scale;                  // bits of the largest |factor|: the result is 2^-14 times this, null: 1
};

__device__ __forceinline__ void tile_at(const Problem &p, int t, int &m, int &n, int &split)
{
    const int tiles = p.m_tiles * p.n_tiles;
    split = t / tiles;
    t -= split * tiles;
    if (p.m_fast) m = t % p.m_tiles, n = t / p.m_tiles;
    else n = t % p.n_tiles, m = t / p.n_tiles;
}

template <class T>
__device__ __forceinline__ void store_columns(T *to, const float (&v)[32], int n)
{
    constexpr int kWide = 16 / sizeof(T);
    if (n == 32 && (uintptr_t)to % 16 == 0) {
#pragma unroll
        for (int j = 0; j < 32; j += kWide) {
            Pack<T, kWide> q;
#pragma unroll
            for (int k = 0; k < kWide; k++) q.v[k] = from_float<T>(v[j + k]);
            *(Pack<T, kWide> *)(to + j) = q;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < n) to[j] = from_float<T>(v[j]);
    }
}

// Softmax statistics of a row, over the 32 products `v` at a time.
struct RowSums {
    float largest = -INFINITY, sum = 0.f;
    __device__ __forceinline__ void take(const float (&v)[32], float slope)
    {
        float top = v[0];
#pragma unroll
        for (int j = 1; j < 32; j++) top = fmaxf(top, v[j]);
        const float next = fmaxf(largest, top), from = next == -INFINITY ? 0.f : next;
        if (largest > -INFINITY) sum *= exp2_fast((largest - from) * slope);
#pragma unroll
        for (int j = 0; j < 32; j++) sum += exp2_fast((v[j] - from) * slope);
        largest = next;
    }
};

// The same with the first largest one's index and without its own 1 in the sum.
struct RowBest {
    float largest = -INFINITY, rest = 0.f;
    int index = -1;
    __device__ __forceinline__ void take(const float (&v)[32], float slope, int first)
    {
        float top = v[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < 32; j++)
            if (v[j] > top || !(top == top)) top = v[j], at = j;
        const float from = top == -INFINITY || !(top == top) ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 32; j++) sum += j == at && top > -INFINITY ? 0.f : exp2_fast((v[j] - from) * slope);
        if (!(top > -INFINITY)) rest += sum;                       // nothing but -inf (sum is 0) or NaN
        else if (top > largest) rest = (largest > -INFINITY ? (rest + 1.f) * exp2_fast((largest - top) * slope) : rest) + sum, largest = top, index = first + at;
        else rest += (sum + 1.f) * exp2_fast((top - largest) * slope);
    }
};

template <int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
softmax_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Problem p)
{
    extern __shared__ unsigned char shared_raw[];
    __shared__ alignas(8) unsigned long long barriers[2 * kStages + 4];
    __shared__ unsigned tmem_shared;
    const unsigned ring = (smem_address(shared_raw) + 1023) & ~1023u;
    const unsigned full = smem_address(barriers), empty = full + 8 * kStages, sums_full = empty + 8 * kStages, sums_empty = sums_full + 16;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const unsigned rank = cluster_rank();
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

    const int tiles = p.m_tiles * p.n_tiles * p.splits, first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;
    const int half_columns = p.tile_columns / 2, all_blocks = p.depth_blocks * p.products;
    bool fine = true;
    if (warp == 0 && lane == 0) {
        // copies: the ring's stages of this block, counted on the leader's barriers
        int stage = 0, phase = 0;
        for (int t = first_tile; t < tiles && fine; t += tile_step) {
            int m, n, split;
            tile_at(p, t, m, n, split);
            const int m0 = m * 256 + (int)rank * 128, n0 = n * p.tile_columns + (int)rank * half_columns + p.b_row;
            const int last = min(all_blocks, (split + 1) * p.per_split);
            for (int i = split * p.per_split; i < last; i++) {
                if (!(fine = barrier_wait(empty + 8 * stage, phase ^ 1))) break;
                const unsigned to = ring + stage * kStageBytes, bar = in_leader(full + 8 * stage);
                if (rank == 0) barrier_expect(full + 8 * stage, 2 * (kHalfBytes + half_columns * kDepth * 2));
                int part_a, part_b;
                parts_of(p.products, i / p.depth_blocks, part_a, part_b);
                const int k = i % p.depth_blocks * kDepth;
                if (p.a_rows)
                    for (int g = 0; g < 2; g++) load_box(&map_a, to + g * 8192, bar, m0 + g * 64, p.a_first + k, part_a);
                else load_box(&map_a, to, bar, p.a_first + k, m0, part_a);
                if (p.b_rows)
                    for (int g = 0; g < half_columns / 64; g++) load_box(&map_b, to + kHalfBytes + g * 8192, bar, n0 + g * 64, p.b_first + k, part_b);
                else load_box(&map_b, to + kHalfBytes, bar, p.b_first + k, n0, part_b);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        }
        // the products' last arrivals come to this block's barriers before it ends
        for (int i = 0; i < kStages && fine; i++) {
            fine = barrier_wait(empty + 8 * stage, phase ^ 1);
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
        // copies that nobody will wait for any more end before the block does: 20 ms are thousands of times what one takes
        if (!fine)
            for (const unsigned long long began = nanoseconds(); nanoseconds() - began < 20000000ull;) __nanosleep(1000);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        int stage = 0, phase = 0, buffer = 0, buffer_phase = 0;
        // rows next to each other: 64 of them and 8 of the sum's index are 1024 bytes, 64 more rows one box further; a step of 16 is 2048 bytes.
        // the sum's index next to each other: 8 rows are 1024 bytes; a step of 16 is 32 bytes
        const unsigned a_leading = p.a_rows ? 8192 : 16, b_leading = p.b_rows ? 8192 : 16, a_step = p.a_rows ? 2048 : 32, b_step = p.b_rows ? 2048 : 32;
        for (int t = first_tile; t < tiles && fine; t += tile_step) {
            int m, n, split;
            tile_at(p, t, m, n, split);
            if (!(fine = barrier_wait(sums_empty + 8 * buffer, buffer_phase ^ 1))) break;
            tmem_after_sync();
            const unsigned to = tmem + buffer * 256;
            const int first = split * p.per_split, last = min(all_blocks, first + p.per_split);
            for (int i = first; i < last; i++) {
                if (!(fine = barrier_wait(full + 8 * stage, phase))) break;
                tmem_after_sync();
                const unsigned a = ring + stage * kStageBytes, b = a + kHalfBytes;
#pragma unroll
                for (int k = 0; k < kDepth / 16; k++)
                    multiply(to, operand(a + k * a_step, a_leading, 1024), operand(b + k * b_step, b_leading, 1024), p.what, i > first || k > 0);
                commit_to_pair(empty + 8 * stage);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
            if (!fine) break;
            commit_to_pair(sums_full + 8 * buffer);
            if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
        }
    } else if (warp >= 4) {
        const int w = (warp - 4) & 3, half = (warp - 4) / 4;
        int buffer = 0, buffer_phase = 0;
        for (int t = first_tile; t < tiles; t += tile_step) {
            int m, n, split;
            tile_at(p, t, m, n, split);
            fine = barrier_wait(sums_full + 8 * buffer, buffer_phase);
            if (!__all_sync(~0u, fine)) break;
            tmem_after_sync();
            const long long row = (long long)m * 256 + rank * 128 + w * 32 + lane;
            const bool real = row < p.rows;
            const unsigned from = tmem + buffer * 256 + half * half_columns + ((unsigned)(w * 32) << 16);
            const long long column0 = (long long)n * p.tile_columns + half * half_columns;
            RowSums sums;
            RowBest best;
            float normaliser = 0.f, factor = 0.f;
            int label = -1;
            if ((kMode == kSums || kMode == kProb) && real && p.labels) label = p.labels[row] - p.first_label;
            if (kMode == kProb && real) {
                normaliser = p.normalisers[row], factor = p.factors[row];
                if (p.largest) {
                    const float largest = __uint_as_float(*p.largest);
                    factor = largest == 0.f ? 0.f : factor / largest * 16384.f;
                }
            }
            const float out_scale = kMode == kOut && p.out_scale ? __uint_as_float(*p.out_scale) * (1.f / 16384.f) : 1.f;
            for (int c = 0; c < half_columns; c += 32) {
                float v[32];
                tmem_load(from + c, v);
                const long long column = column0 + c, left = p.columns - column;
                if (left <= 0) continue;                                    // the warp together
                if (kMode == kSums || kMode == kBest) {
                    if (left < 32)
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (j >= left) v[j] = -INFINITY;
                    if (kMode == kSums) {
                        sums.take(v, p.scale * kLog2e);
                        const long long at = label - column;
                        if (__any_sync(~0u, at >= 0 && at < 32 && label >= 0)) {
                            float mine = 0.f;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (at == j) mine = v[j];
                            if (label >= 0 && at >= 0 && at < 32 && real) p.label_logit[row] = mine;
                        }
                    } else {
                        best.take(v, p.scale * kLog2e, (int)column);
                    }
                } else if (kMode == kProb) {
                    const long long at = label - column;
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        float q = exp2_fast(fmaf(v[j], p.scale, -normaliser) * kLog2e);
                        if (at == j) q -= 1.f;
                        v[j] = factor == 0.f ? 0.f : q * factor;
                    }
                    if (real) {
                        const long long to = row * p.prob_stride + column;
                        if (p.type == GTM_F16) store_columns((__half *)p.prob + to, v, 32);
                        else {
                            store_columns((__nv_bfloat16 *)p.prob + to, v, 32);
                            if (p.products > 1)
                                for (int part = 1; part < 3; part++) {
#pragma unroll
                                    for (int j = 0; j < 32; j++) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
                                    store_columns((__nv_bfloat16 *)p.prob + part * p.prob_part + to, v, 32);
                                }
                        }
                    }
                } else if (real) {
                    const int n_left = left < 32 ? (int)left : 32;
                    if (p.partial) {
                        float *to = p.partial + (split * p.rows + row) * p.columns + column;
                        if (p.add)
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (j < n_left) v[j] += to[j];
                        store_columns(to, v, n_left);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] *= out_scale;
                        const long long to = row * p.out_stride + column;
                        if (p.type == GTM_F32) store_columns((float *)p.out + to, v, n_left);
                        else if (p.type == GTM_F16) store_columns((__half *)p.out + to, v, n_left);
                        else store_columns((__nv_bfloat16 *)p.out + to, v, n_left);
                    }
                }
            }
            if ((kMode == kSums || kMode == kBest) && real) {
                const long long at = (n * 2ll + half) * p.rows + row;
                p.sums[at] = kMode == kSums ? make_float2(sums.largest, sums.sum) : make_float2(best.largest, best.rest);
                if (kMode == kBest) p.best[at] = best.index;
            }
            tmem_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive_leader(in_leader(sums_empty + 8 * buffer));
            if (++buffer == 2) buffer = 0, buffer_phase ^= 1;
        }
    }
    if (!fine) atomicExch(p.error, 1);
    __syncwarp();
    tmem_before_sync();
    cluster_sync();
    tmem_after_sync();
    if (warp == 2) tmem_free(tmem, 512);
}

// ------------------------------------------------------------------------------------------- around the products
// Rows of a matrix with 16-byte boundaries, in parts where they are 32-bit ones; rows of examples that are ignored are zero.
template <class T>
__global__ void __launch_bounds__(256) softmax_lay_out_kernel(const T *from, long long stride, long long rows, int columns, const int *labels, void *to, long long to_stride, long long part)
{
    const long long all = rows * columns;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long r = i / columns, c = i - r * columns;
        const bool kept = !labels || labels[r] != -1;
        if constexpr (sizeof(T) == 4) {
            float v = kept ? from[r * stride + c] : 0.f;
            __nv_bfloat16 *q = (__nv_bfloat16 *)to + r * to_stride + c;
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const __nv_bfloat16 b = __float2bfloat16_rn(v);
                q[k * part] = b;
                v = fabsf(__bfloat162float(b)) <= 3.4e38f ? v - __bfloat162float(b) : 0.f;
            }
        } else {
            ((T *)to)[r * to_stride + c] = kept ? from[r * stride + c] : from_float<T>(0.f);
        }
    }
}

// Labels as 32 bits: -1 for ignored examples, -2 for labels that there are not.  With gradients: the factor of every row of P.
__global__ void __launch_bounds__(256) softmax_rows_kernel(const void *labels, int labels_64, long long rows, long long number_of_labels, long long ignored, const float *gradients,
                                                           int gradients_step, float scale, int *out, float *factors, unsigned *largest)
{
    const long long r = (long long)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const long long l = index_at(labels, labels_64, r);
    const int label = l == ignored ? -1 : l < 0 || l >= number_of_labels ? -2 : (int)l;
    out[r] = label;
    if (!factors) return;
    const float f = label == -1 ? 0.f : label == -2 ? __int_as_float(0x7fffffff) : gradients[r * gradients_step] * scale;
    factors[r] = f;
    if (largest) atomicMax(largest, __float_as_uint(fabsf(f)));      // of magnitudes: the bits have their order, NaN above all
}

// Joins the parts of 32 rows; a row's parts are read by 32 threads.
__global__ void __launch_bounds__(1024) softmax_loss_kernel(const float2 *sums, const float *label_logit, const int *labels, long long rows, int parts, float scale, float *losses,
                                                            float *normalisers)
{
    __shared__ float tops[32][33], all[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x / 32;
    const long long row = (long long)blockIdx.x * 32 + x;
    float top = -INFINITY, sum = 0.f;
    const auto join = [&](float t, float s) {
        const float next = fmaxf(top, t);
        if (next == -INFINITY) { sum += s; return; }
        sum = (top == -INFINITY ? sum : sum * expf((top - next) * scale)) + (t == -INFINITY ? s : s * expf((t - next) * scale));
        top = next;
    };
    if (row < rows)
        for (int i = y; i < parts; i += 32) {
            const float2 s = sums[(long long)i * rows + row];
            join(s.x, s.y);
        }
    tops[y][x] = top, all[y][x] = sum;
    __syncthreads();
    // a warp joins one row's 32
    const long long mine = (long long)blockIdx.x * 32 + y;
    top = tops[x][y], sum = all[x][y];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const float t = __shfl_xor_sync(~0u, top, o), s = __shfl_xor_sync(~0u, sum, o);
        join(t, s);
    }
    if (x || mine >= rows) return;
    const float log_sum = logf(sum);
    normalisers[mine] = fmaf(top, scale, log_sum);
    if (losses) {
        const int label = labels[mine];
        losses[mine] = label == -1 ? 0.f : label == -2 ? __int_as_float(0x7fffffff) : fmaf(top - label_logit[mine], scale, log_sum);
    }
}

__global__ void __launch_bounds__(1024) softmax_best_kernel(const float2 *sums, const int *best, long long rows, int parts, float scale, long long *labels, float *log_probabilities)
{
    __shared__ float tops[32][33], all[32][33];
    __shared__ int indices[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x / 32;
    const long long row = (long long)blockIdx.x * 32 + x;
    float top = -INFINITY, rest = 0.f;
    int index = 0x7fffffff;
    const auto join = [&](float t, float r, int i) {
        if (t == -INFINITY) { rest += r; return; }
        if (top == -INFINITY) { top = t, rest += r, index = i; return; }
        const bool other = t > top || (t == top && i < index);
        const float high = other ? t : top, low = other ? top : t;
        rest = (other ? r : rest) + (1.f + (other ? rest : r)) * expf((low - high) * scale);
        top = high, index = other ? i : index;
    };
    if (row < rows)
        for (int i = y; i < parts; i += 32) {
            const float2 s = sums[(long long)i * rows + row];
            join(s.x, s.y, best[(long long)i * rows + row]);
        }
    tops[y][x] = top, all[y][x] = rest, indices[y][x] = index;
    __syncthreads();
    const long long mine = (long long)blockIdx.x * 32 + y;
    top = tops[x][y], rest = all[x][y], index = indices[x][y];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const float t = __shfl_xor_sync(~0u, top, o), r = __shfl_xor_sync(~0u, rest, o);
        const int i = __shfl_xor_sync(~0u, index, o);
        join(t, r, i);
    }
    if (x || mine >= rows) return;
    const float log_probability = top == -INFINITY ? __int_as_float(0x7fffffff) : -log1pf(rest);
    log_probabilities[mine] = log_probability;
    labels[mine] = log_probability == log_probability ? index : -1;
}

// Adds the slices of a product up, in their order.
template <class T>
__global__ void __launch_bounds__(256) softmax_finish_kernel(const float *partial, int slices, long long rows, int columns, const unsigned *out_scale, T *out, long long stride)
{
    const float factor = out_scale ? __uint_as_float(*out_scale) * (1.f / 16384.f) : 1.f;
    const long long all = rows * columns;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        float sum = 0.f;
        for (int s = 0; s < slices; s++) sum += partial[s * all + i];
        out[i / columns * stride + i % columns] = from_float<T>(sum * factor);
    }
}

// -------------------------------------------------------------------------------------------------------- host side
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_tiled(EncodeTiled *out)
{
    static EncodeTiled found = nullptr;          // the same whichever thread finds it
    if (!found) {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult result;
        GTM_CU(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result));
        if (result != cudaDriverEntryPointSuccess || !f) return fail(GTM_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        found = (EncodeTiled)f;
    }
    *out = found;
    return GTM_OK;
}

// A matrix as the kernels read it: rows at 16-byte boundaries, one part or three.
struct Matrix {
    const void *data;
    int64_t rows, columns, stride, part;         // elements
    int parts;
    bool fp16;
};

int make_map(CUtensorMap *map, const Matrix &a, unsigned box_columns, unsigned box_rows)
{
    EncodeTiled encode;
    GTM_TRY(encode_tiled(&encode));
    const cuuint64_t sizes[3] = {(cuuint64_t)a.columns, (cuuint64_t)a.rows, (cuuint64_t)a.parts};
    const cuuint64_t strides[2] = {(cuuint64_t)a.stride * 2, (cuuint64_t)(a.parts > 1 ? a.part : a.stride * a.rows) * 2};
    const cuuint32_t box[3] = {box_columns, box_rows, 1}, steps[3] = {1, 1, 1};
    const CUresult r = encode(map, a.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void *)a.data, sizes, strides, box, steps,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GTM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %lld x %lld elements, stride %lld", (int)r, (long long)a.rows, (long long)a.columns, (long long)a.stride);
    return GTM_OK;
}

__device__ int softmax_error;                    // set by a wait that ran out

template <int kMode>
int launch_product(Problem p, const Matrix &a, const Matrix &b, cudaStream_t stream)
{
    CUtensorMap map_a, map_b;
    GTM_TRY(make_map(&map_a, a, 64, p.a_rows ? 64 : 128));
    GTM_TRY(make_map(&map_b, b, 64, p.b_rows ? 64 : p.tile_columns / 2));
    p.what = product(a.fp16 ? 0 : 1, p.tile_columns, p.a_rows, p.b_rows);
    void *error = nullptr;
    GTM_CU(cudaGetSymbolAddress(&error, softmax_error));
    p.error = (int *)error;
    GTM_CU(cudaFuncSetAttribute(softmax_product_kernel<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared));
    int device = 0, sms = 0;
    GTM_CU(cudaGetDevice(&device));
    GTM_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    const int tiles = p.m_tiles * p.n_tiles * p.splits;
    softmax_product_kernel<kMode><<<2 * std::min(tiles, sms / 2), kThreads, kShared, stream>>>(map_a, map_b, p);
    GTM_CU(cudaGetLastError());
    return GTM_OK;
}

// Tiles of 128 columns where 256 would leave pairs of SMs without one.
int tile_columns(int64_t rows, int64_t columns)
{
    return columns <= 128 || (rows + 255) / 256 * ((columns + 255) / 256) < kPairs ? 128 : 256;
}

struct Shape {
    int m_tiles, n_tiles, tile, splits, per_split, depth_blocks;
};

// Tiles of a product; where they are fewer than the pairs of SMs, the sum's index is split, into eight blocks or more.
Shape shape_of(int64_t rows, int64_t columns, int64_t depth, int products, bool split)
{
    Shape s;
    s.tile = tile_columns(rows, columns);
    s.m_tiles = (int)((rows + 255) / 256), s.n_tiles = (int)((columns + s.tile - 1) / s.tile);
    s.depth_blocks = (int)((depth + kDepth - 1) / kDepth);
    const int blocks = s.depth_blocks * products, tiles = s.m_tiles * s.n_tiles;
    s.splits = split ? std::max(1, std::min(kPairs / tiles, blocks / 8)) : 1;
    s.per_split = (blocks + s.splits - 1) / s.splits;
    s.splits = (blocks + s.per_split - 1) / s.per_split;
    return s;
}

Problem problem_of(const Shape &s, int64_t rows, int64_t columns, int products)
{
    Problem p = {};
    p.rows = rows, p.columns = columns, p.m_tiles = s.m_tiles, p.n_tiles = s.n_tiles, p.splits = s.splits, p.tile_columns = s.tile;
    p.depth_blocks = s.depth_blocks, p.per_split = s.per_split, p.products = products;
    return p;
}

// What a call reads, and where its workspace's parts are.
struct Call {
    int type, products, parts;
    int64_t examples, labels, columns;
    const void *x, *w;
    int64_t x_stride, w_stride;
    bool lay_out_x, lay_out_w, gradient;
    int64_t x_ld, w_ld;
    // forward
    int64_t piece_rows;
    int stat_parts;
    // gradient
    int64_t piece_labels, prob_ld;
    Shape dx, dw;
    bool dx_partial, dw_partial;
    uint64_t at_x, at_w, at_rows, at_factors, at_largest, at_sums, at_best, at_logit, at_prob, at_dx, at_dw, total;
};

bool direct(int type, const void *p, int64_t rows, int64_t stride, int64_t columns)
{
    return type != GTM_F32 && (uintptr_t)p % 16 == 0 && (rows == 1 || (stride * 2 % 16 == 0 && stride >= columns));
}

int64_t clamp64(int64_t v, int64_t low, int64_t high) { return v < low ? low : v > high ? high : v; }

void lay_out_workspace(Call &c)
{
    c.products = c.type == GTM_F32 ? kPartProducts : 1;
    c.parts = c.type == GTM_F32 ? 3 : 1;
    // the gradient's x is laid out anew in any case: examples that are ignored may hold anything
    c.lay_out_x = c.gradient || !direct(c.type, c.x, c.examples, c.x_stride, c.columns);
    c.lay_out_w = !direct(c.type, c.w, c.labels, c.w_stride, c.columns);
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
        c.stat_parts = (int)((c.labels + tile - 1) / tile) * 2;
        c.piece_rows = std::min<int64_t>(c.examples, clamp64(kStatBytes / (c.stat_parts * 8) / 256 * 256, 256, (int64_t)1 << 30));
        c.at_sums = take((uint64_t)c.stat_parts * c.piece_rows * 8);
        c.at_best = take((uint64_t)c.stat_parts * c.piece_rows * 4);
        c.at_logit = take(c.piece_rows * 4);
    } else {
        c.at_factors = take(c.examples * 4);
        c.at_largest = take(4);
        const int64_t most = clamp64(kPieceBytes / (c.examples * 2 * c.parts) / 256 * 256, 256, (int64_t)1 << 30);
        const int64_t pieces = (c.labels + most - 1) / most;
        c.piece_labels = pieces == 1 ? c.labels : (int64_t)round_up((c.labels + pieces - 1) / pieces, 256);
        c.prob_ld = (int64_t)round_up(c.piece_labels, 64);
        c.at_prob = take((uint64_t)c.parts * c.examples * c.prob_ld * 2);
        c.dx = shape_of(c.examples, c.columns, c.piece_labels, c.products, true);
        c.dw = shape_of(c.piece_labels, c.columns, c.examples, c.products, true);
        c.dx_partial = c.dx.splits > 1 || pieces > 1;
        c.dw_partial = c.dw.splits > 1;
        c.at_dx = take(c.dx_partial ? (uint64_t)c.dx.splits * c.examples * c.columns * 4 : 0);
        c.at_dw = take(c.dw_partial ? (uint64_t)c.dw.splits * c.piece_labels * c.columns * 4 : 0);
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
void lay_out(const void *from, int64_t stride, int64_t rows, int64_t columns, const int *labels, void *to, int64_t ld, cudaStream_t stream)
{
    const int64_t blocks = std::min<int64_t>((rows * columns + 255) / 256, 148 * 16);
    softmax_lay_out_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>((const T *)from, stride, rows, (int)columns, labels, to, ld, rows * ld);
}

// A matrix as the kernels read it, laid out in the workspace where it is not so already.
int operand_of(Matrix *out, int type, const void *data, int64_t stride, int64_t rows, int64_t columns, bool copy, const int *labels, void *to, int64_t ld, cudaStream_t stream)
{
    if (copy) {
        if (type == GTM_F32) lay_out<float>(data, stride, rows, columns, labels, to, ld, stream);
        else if (type == GTM_BF16) lay_out<__nv_bfloat16>(data, stride, rows, columns, labels, to, ld, stream);
        else lay_out<__half>(data, stride, rows, columns, labels, to, ld, stream);
        GTM_CU(cudaGetLastError());
        data = to;
    }
    *out = {data, rows, columns, ld, rows * ld, type == GTM_F32 ? 3 : 1, type == GTM_F16};
    return GTM_OK;
}

int finish(int type, const float *partial, int slices, int64_t rows, int64_t columns, const unsigned *out_scale, void *out, int64_t stride, cudaStream_t stream)
{
    const unsigned blocks = (unsigned)std::min<int64_t>((rows * columns + 255) / 256, 148 * 16);
    if (type == GTM_F32) softmax_finish_kernel<float><<<blocks, 256, 0, stream>>>(partial, slices, rows, (int)columns, out_scale, (float *)out, stride);
    else if (type == GTM_BF16) softmax_finish_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(partial, slices, rows, (int)columns, out_scale, (__nv_bfloat16 *)out, stride);
    else softmax_finish_kernel<__half><<<blocks, 256, 0, stream>>>(partial, slices, rows, (int)columns, out_scale, (__half *)out, stride);
    GTM_CU(cudaGetLastError());
    return GTM_OK;
}

// Loss (labels given) or most probable label.
int forward(const char *what, Call &c, const void *labels, int labels_64, int64_t ignored, float scale, float *losses, float *normalisers, int64_t *best, float *log_probabilities,
            char *w, cudaStream_t stream)
{
    Matrix x, weights;
    int *rows = labels ? (int *)(w + c.at_rows) : nullptr;
    if (labels) {
        softmax_rows_kernel<<<(unsigned)((c.examples + 255) / 256), 256, 0, stream>>>(labels, labels_64, c.examples, c.labels, ignored, nullptr, 0, scale, rows, nullptr, nullptr);
        GTM_CU(cudaGetLastError());
    }
    GTM_TRY(operand_of(&x, c.type, c.x, c.x_stride, c.examples, c.columns, c.lay_out_x, nullptr, w + c.at_x, c.x_ld, stream));
    GTM_TRY(operand_of(&weights, c.type, c.w, c.w_stride, c.labels, c.columns, c.lay_out_w, nullptr, w + c.at_w, c.w_ld, stream));
    for (int64_t r = 0; r < c.examples; r += c.piece_rows) {
        const int64_t n = std::min(c.piece_rows, c.examples - r);
        Matrix piece = x;
        piece.data = (const char *)x.data + r * x.stride * 2;
        piece.rows = n;
        Shape s = shape_of(n, c.labels, c.columns, c.products, false);
        s.tile = tile_columns(c.examples, c.labels);         // as the workspace has it
        s.n_tiles = (int)((c.labels + s.tile - 1) / s.tile);
        Problem p = problem_of(s, n, c.labels, c.products);
        p.m_fast = 1, p.scale = scale, p.sums = (float2 *)(w + c.at_sums), p.best = (int *)(w + c.at_best), p.label_logit = (float *)(w + c.at_logit);
        p.labels = labels ? rows + r : nullptr;
        const unsigned blocks = (unsigned)((n + 31) / 32);
        if (labels) {
            GTM_TRY(launch_product<kSums>(p, piece, weights, stream));
            softmax_loss_kernel<<<blocks, 1024, 0, stream>>>(p.sums, p.label_logit, rows + r, n, s.n_tiles * 2, scale, losses + r, normalisers + r);
        } else {
            GTM_TRY(launch_product<kBest>(p, piece, weights, stream));
            softmax_best_kernel<<<blocks, 1024, 0, stream>>>(p.sums, p.best, n, s.n_tiles * 2, scale, (long long *)best + r, log_probabilities + r);
        }
        GTM_CU(cudaGetLastError());
    }
    return GTM_OK;
}

}  // namespace
}  // namespace gtm_readout

using namespace gtm_readout;

static Call call_of(int type, int64_t examples, int64_t labels, int64_t columns, const void *x, int64_t x_stride, const void *w, int64_t w_stride, bool gradient)
{
    Call c = {};
    c.type = type, c.examples = examples, c.labels = labels, c.columns = columns, c.x = x, c.w = w, c.x_stride = x_stride, c.w_stride = w_stride, c.gradient = gradient;
    return c;
}

extern "C" int gtm_softmax_workspace(int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t labels, int64_t weights_stride,
                                     int64_t columns, int gradient, uint64_t *bytes_out)
{
    if (!bytes_out) return fail(GTM_ERR_ARG, "gtm_softmax_workspace: null output");
    Call c = call_of(type, examples, labels, columns, features, features_stride, weights, weights_stride, gradient != 0);
    GTM_TRY(check_call("gtm_softmax_workspace", c, 1.f));
    *bytes_out = 0;
    if (examples == 0) return GTM_OK;
    lay_out_workspace(c);
    *bytes_out = c.total;
    return GTM_OK;
}

extern "C" int gtm_softmax_loss(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t number_of_labels,
                                int64_t weights_stride, int64_t columns, const void *labels, int labels_64, int64_t ignore_label, float scale, float *losses, float *normalisers,
                                void *workspace, uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, false);
    GTM_TRY(check_call("gtm_softmax_loss", c, scale));
    if (examples == 0) return GTM_OK;
    if (!features || !weights || !labels || !losses || !normalisers) return fail(GTM_ERR_ARG, "gtm_softmax_loss: null array");
    lay_out_workspace(c);
    GTM_TRY(check_workspace("gtm_softmax_loss", workspace, workspace_bytes, c.total));
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    return forward("gtm_softmax_loss", c, labels, labels_64, ignore_label, scale, losses, normalisers, nullptr, nullptr, (char *)workspace, (cudaStream_t)cuda_stream);
}

extern "C" int gtm_softmax_predict(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights, int64_t number_of_labels,
                                   int64_t weights_stride, int64_t columns, float scale, int64_t *labels_out, float *log_probabilities_out, void *workspace, uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, false);
    GTM_TRY(check_call("gtm_softmax_predict", c, scale));
    if (examples == 0) return GTM_OK;
    if (!features || !weights || !labels_out || !log_probabilities_out) return fail(GTM_ERR_ARG, "gtm_softmax_predict: null array");
    lay_out_workspace(c);
    GTM_TRY(check_workspace("gtm_softmax_predict", workspace, workspace_bytes, c.total));
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    return forward("gtm_softmax_predict", c, nullptr, 0, 0, scale, nullptr, nullptr, labels_out, log_probabilities_out, (char *)workspace, (cudaStream_t)cuda_stream);
}

extern "C" int gtm_softmax_loss_gradient(int device, void *cuda_stream, int type, const void *features, int64_t examples, int64_t features_stride, const void *weights,
                                         int64_t number_of_labels, int64_t weights_stride, int64_t columns, const void *labels, int labels_64, int64_t ignore_label, float scale,
                                         const float *normalisers, const float *gradients, int64_t gradients_step, void *features_gradient, int64_t features_gradient_stride,
                                         void *weights_gradient, int64_t weights_gradient_stride, void *workspace, uint64_t workspace_bytes)
{
    Call c = call_of(type, examples, number_of_labels, columns, features, features_stride, weights, weights_stride, true);
    GTM_TRY(check_call("gtm_softmax_loss_gradient", c, scale));
    if (!weights_gradient || weights_gradient_stride < columns || (examples && features_gradient_stride < columns))
        return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: null result or a row stride below its columns");
    if (gradients_step != 0 && gradients_step != 1) return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: step %lld of the gradients (0 or 1)", (long long)gradients_step);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    if (examples == 0) {
        GTM_CU(cudaMemset2DAsync(weights_gradient, weights_gradient_stride * type_bytes(type), 0, columns * type_bytes(type), number_of_labels, stream));
        return GTM_OK;
    }
    if (!features || !weights || !labels || !normalisers || !gradients || !features_gradient) return fail(GTM_ERR_ARG, "gtm_softmax_loss_gradient: null array");
    lay_out_workspace(c);
    GTM_TRY(check_workspace("gtm_softmax_loss_gradient", workspace, workspace_bytes, c.total));
    char *w = (char *)workspace;
    int *rows = (int *)(w + c.at_rows);
    float *factors = (float *)(w + c.at_factors);
    unsigned *largest = type == GTM_F16 ? (unsigned *)(w + c.at_largest) : nullptr;
    if (largest) GTM_CU(cudaMemsetAsync(largest, 0, 4, stream));
    softmax_rows_kernel<<<(unsigned)((examples + 255) / 256), 256, 0, stream>>>(labels, labels_64, examples, number_of_labels, ignore_label, gradients, (int)gradients_step, scale, rows, factors, largest);
    GTM_CU(cudaGetLastError());
    Matrix x, wm;
    GTM_TRY(operand_of(&x, type, features, features_stride, examples, columns, true, rows, w + c.at_x, c.x_ld, stream));
    GTM_TRY(operand_of(&wm, type, weights, weights_stride, number_of_labels, columns, c.lay_out_w, nullptr, w + c.at_w, c.w_ld, stream));
    float *dx = c.dx_partial ? (float *)(w + c.at_dx) : nullptr, *dw = c.dw_partial ? (float *)(w + c.at_dw) : nullptr;
    for (int64_t v = 0; v < number_of_labels; v += c.piece_labels) {
        const int64_t n = std::min(c.piece_labels, number_of_labels - v);
        const Matrix prob = {w + c.at_prob, examples, n, c.prob_ld, examples * c.prob_ld, c.parts, type == GTM_F16};
        // P of the piece
        Matrix piece = wm;                        // rows behind the piece read as zeros
        piece.rows = v + n;
        Problem p = problem_of(shape_of(examples, n, columns, c.products, false), examples, n, c.products);
        p.m_fast = 1, p.b_row = (int)v, p.scale = scale, p.labels = rows, p.first_label = (int)v;
        p.normalisers = normalisers, p.factors = factors, p.largest = largest, p.type = type;
        p.prob = (void *)prob.data, p.prob_stride = c.prob_ld, p.prob_part = prob.part;
        GTM_TRY(launch_product<kProb>(p, x, piece, stream));
        // dw of the piece: sums over examples
        Shape s = shape_of(n, columns, examples, c.products, false);
        s.splits = c.dw.splits, s.per_split = c.dw.per_split;       // as the workspace has them, for a smaller last piece too
        p = problem_of(s, n, columns, c.products);
        p.a_rows = p.b_rows = 1, p.type = type, p.out_scale = largest, p.partial = dw;
        p.out = (char *)weights_gradient + v * weights_gradient_stride * type_bytes(type), p.out_stride = weights_gradient_stride;
        GTM_TRY(launch_product<kOut>(p, prob, x, stream));
        if (dw) GTM_TRY(finish(type, dw, p.splits, n, columns, largest, p.out, p.out_stride, stream));
        // dx: sums over the piece's labels
        p = problem_of(c.dx, examples, columns, c.products);
        p.b_rows = 1, p.b_first = (int)v, p.type = type, p.out_scale = largest, p.partial = dx, p.add = v > 0;
        p.out = features_gradient, p.out_stride = features_gradient_stride;
        GTM_TRY(launch_product<kOut>(p, prob, piece, stream));
    }
    if (dx) GTM_TRY(finish(type, dx, c.dx.splits, examples, columns, largest, features_gradient, features_gradient_stride, stream));
    return GTM_OK;
}

extern "C" int gtm_softmax_failed(int device, int *failed_out)
{
    if (!failed_out) return fail(GTM_ERR_ARG, "gtm_softmax_failed: null output");
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    const int zero = 0;
    GTM_CU(cudaDeviceSynchronize());
    GTM_CU(cudaMemcpyFromSymbol(failed_out, softmax_error, sizeof(int)));
    GTM_CU(cudaMemcpyToSymbol(softmax_error, &zero, sizeof(int)));
    return GTM_OK;
}
