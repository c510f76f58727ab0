// Softmax cross entropy, its gradient and the most probable label where there are at most 32 labels: a machine's classes.
//
// The weights fit in shared memory, in 32 bits, and a warp has two examples at a time: its lanes hold the columns for the dot products and
// then a label each.  One launch for the forward pass.  The gradient's first launch computes the logits again, dx, and each
// block's sums of dw over its examples (P in shared memory, a thread per column); the second adds the blocks' sums up, in their order.
// What bounds it is the number of launches and, for many examples, reading x; the tensor cores' tiles would be mostly empty: 60 examples of 64
// columns and ten labels in 32 bits take 4 us forward and 9 for the gradient, where products by tiles took 20 and 45.  Loss and gradient take the same
// logits, those of these kernels, for as many examples: where P of the label is near one, a logit's error leaves it with the normaliser.  Up to 2^16 examples, whose P a block has
// in 28 KB of shared memory; for more, tiles are faster (66,000 examples of 512 bf16, 32 labels: 48 and 1,110 us for loss and gradient, 163 and 1,920 with
// these kernels and their examples in pieces; of 64 bf16, ten labels: 42 and 99 instead of 45 and 151).
#include "gtm_readout.cuh"
#include "gtm_readout_softmax.h"

#include <algorithm>

namespace gtm_readout {
namespace {

constexpr int kWarps = 8, kTogether = 2;                // warps of a block, examples that a warp has at a time
constexpr int kLargestShared = 96 << 10;                // bytes of weights

struct Args {
    FewLabels p;
    int per_block;                                      // examples
    float *losses, *normalisers_out;
    long long *labels_out;
    float *log_probabilities;
    const float *normalisers, *gradients;
    int gradients_step;
    void *dx;
    float *partial;                                     // [block][label][column]
};

__device__ __forceinline__ float sum_of(float v)
{
#pragma unroll
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

__device__ __forceinline__ float max_of(float v)
{
#pragma unroll
    for (int o = 16; o; o /= 2) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// Label of an example: -1 ignored, -2 one that there is not.
__device__ __forceinline__ int label_of(const FewLabels &p, long long example)
{
    const long long l = index_at(p.wanted, p.wanted_64, example);
    return l == p.ignored ? -1 : l < 0 || l >= p.labels ? -2 : (int)l;
}

enum Mode { kLoss, kPredict, kGradient };

template <class T, int kLabels, int kMode>
__global__ void __launch_bounds__(kWarps * 32) few_labels_kernel(const Args a)
{
    next_may_start();
    wait_for_previous();
    extern __shared__ float shared[];
    const FewLabels &p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, columns = (int)p.columns, labels = (int)p.labels;
    float *w = shared;                                   // [label][column]
    float *prob = shared + labels * columns;             // [example of the block][kLabels], kGradient
    for (int v = warp; v < labels; v += kWarps)
        for (int c = lane; c < columns; c += 32) w[v * columns + c] = to_float(((const T *)p.w)[v * p.w_stride + c]);
    __syncthreads();
    const long long first = (long long)blockIdx.x * a.per_block, last = min(first + a.per_block, (long long)p.examples);
    for (long long e0 = first + warp * kTogether; e0 < last; e0 += kWarps * kTogether) {
        float dot[kTogether][kLabels];
        const T *row[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; k++) {
            row[k] = (const T *)p.x + min(e0 + k, last - 1) * p.x_stride;
#pragma unroll
            for (int v = 0; v < kLabels; v++) dot[k][v] = 0.f;
        }
#pragma unroll 2
        for (int c = lane; c < columns; c += 32) {
            float x[kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; k++) x[k] = to_float(row[k][c]);
#pragma unroll
            for (int v = 0; v < kLabels; v++)
                if (v < labels) {
                    const float weight = w[v * columns + c];
#pragma unroll
                    for (int k = 0; k < kTogether; k++) dot[k][v] = fmaf(x[k], weight, dot[k][v]);
                }
        }
#pragma unroll
        for (int k = 0; k < kTogether; k++) {
            const long long e = e0 + k;
            float mine = 0.f;                            // the product of the lane's label
#pragma unroll
            for (int v = 0; v < kLabels; v++) {
                const float all = sum_of(dot[k][v]);
                if (lane == v) mine = all;
            }
            if (e >= last) continue;                     // the warp together
            const bool real = lane < labels;
            if (kMode == kGradient) {
                const int label = label_of(p, e);
                float q = 0.f;
                if (real && label != -1) {
                    q = expf(fmaf(mine, p.scale, -a.normalisers[e]));
                    if (label == lane) q -= 1.f;
                    q = label == -2 ? __int_as_float(0x7fffffff) : q * (a.gradients[e * a.gradients_step] * p.scale);
                }
                if (lane < kLabels) prob[(e - first) * kLabels + lane] = q;
                __syncwarp();
                T *dx = (T *)a.dx + e * columns;
                for (int c = lane; c < columns; c += 32) {
                    float sum = 0.f;
#pragma unroll
                    for (int v = 0; v < kLabels; v++)
                        if (v < labels) sum = fmaf(prob[(e - first) * kLabels + v], w[v * columns + c], sum);
                    dx[c] = from_float<T>(label == -1 ? 0.f : sum);
                }
                continue;
            }
            const float top = max_of(real ? mine : -INFINITY);
            const float from = top == -INFINITY ? 0.f : top;
            const float power = real ? expf((mine - from) * p.scale) : 0.f;
            if (kMode == kLoss) {
                const int label = label_of(p, e);
                const float log_sum = logf(sum_of(power)), wanted = __shfl_sync(~0u, mine, label < 0 ? 0 : label);
                if (lane == 0) {
                    a.normalisers_out[e] = fmaf(top, p.scale, log_sum);
                    a.losses[e] = label == -1 ? 0.f : label == -2 ? __int_as_float(0x7fffffff) : fmaf(top - wanted, p.scale, log_sum);
                }
            } else {
                // all but the first of the largest; a product that is no number makes the sum none
                const unsigned largest = __ballot_sync(~0u, real && mine == top);
                const int best = largest ? __ffs(largest) - 1 : -1;
                const float rest = sum_of(real && lane != best ? (mine == mine ? power : mine) : 0.f);
                if (lane == 0) {
                    const float log_probability = best < 0 || top == -INFINITY ? __int_as_float(0x7fffffff) : -log1pf(rest);
                    a.log_probabilities[e] = log_probability;
                    a.labels_out[e] = log_probability == log_probability ? best : -1;
                }
            }
        }
    }
    if (kMode != kGradient) return;
    __syncthreads();
    // the block's sums of dw: a thread has a column
    for (int c = threadIdx.x; c < columns; c += kWarps * 32) {
        float sum[kLabels];
#pragma unroll
        for (int v = 0; v < kLabels; v++) sum[v] = 0.f;
#pragma unroll 4
        for (long long e = first; e < last; e++) {
            if (label_of(p, e) == -1) continue;          // its features may be anything
            const float x = to_float(((const T *)p.x)[e * p.x_stride + c]);
#pragma unroll
            for (int v = 0; v < kLabels; v++) sum[v] = fmaf(prob[(e - first) * kLabels + v], x, sum[v]);
        }
#pragma unroll
        for (int v = 0; v < kLabels; v++)
            if (v < labels) a.partial[((long long)blockIdx.x * labels + v) * columns + c] = sum[v];
    }
}

// A warp adds 32 sums of dw up over the blocks, its lanes' columns side by side.
template <class T>
__global__ void __launch_bounds__(256) few_labels_join_kernel(const float *partial, int blocks, long long size, T *dw)
{
    next_may_start();
    wait_for_previous();
    const long long i = (long long)blockIdx.x * 32 + (threadIdx.x & 31);
    __shared__ float sums[kWarps][32];
    const int warp = threadIdx.x / 32;
    float sum = 0.f;
    if (i < size)
#pragma unroll 4
        for (int b = warp; b < blocks; b += kWarps) sum += partial[b * size + i];
    sums[warp][threadIdx.x & 31] = sum;
    __syncthreads();
    if (warp || i >= size) return;
    for (int k = 1; k < kWarps; k++) sum += sums[k][threadIdx.x];
    dw[i] = from_float<T>(sum);
}

// Examples of a block: a round of its warps, more only where that would be more than two blocks an SM.
int per_block(int64_t examples)
{
    const int64_t round = kWarps * kTogether, most = 148 * 2;
    return (int)((std::max<int64_t>(1, (examples + round * most - 1) / (round * most))) * round);
}

template <class T, int kLabels, int kMode>
int run(const Args &a, unsigned blocks, cudaStream_t stream)
{
    const size_t shared = (size_t)a.p.labels * a.p.columns * 4 + (kMode == kGradient ? (size_t)a.per_block * kLabels * 4 : 0);
    if (shared > 48 << 10) GTM_CU(cudaFuncSetAttribute(few_labels_kernel<T, kLabels, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kLargestShared));
    return launch_early(few_labels_kernel<T, kLabels, kMode>, dim3(blocks), dim3(kWarps * 32), shared, stream, a);
}

template <class T, int kMode>
int run(const Args &a, unsigned blocks, cudaStream_t stream)
{
    return a.p.labels <= 4 ? run<T, 4, kMode>(a, blocks, stream) : a.p.labels <= 12 ? run<T, 12, kMode>(a, blocks, stream) : run<T, 32, kMode>(a, blocks, stream);
}

template <int kMode>
int run(Args &a, cudaStream_t stream)
{
    a.per_block = per_block(a.p.examples);
    const unsigned blocks = (unsigned)((a.p.examples + a.per_block - 1) / a.per_block);
    return a.p.type == GTM_F32    ? run<float, kMode>(a, blocks, stream)
           : a.p.type == GTM_BF16 ? run<__nv_bfloat16, kMode>(a, blocks, stream)
                                  : run<__half, kMode>(a, blocks, stream);
}

}  // namespace

bool few_labels(int64_t examples, int64_t labels, int64_t columns)
{
    return labels <= 32 && labels * columns * 4 <= kLargestShared && examples <= kFewLabelsExamples;
}

uint64_t few_labels_workspace(int64_t examples, int64_t labels, int64_t columns, bool gradient)
{
    const int64_t each = per_block(examples), blocks = (examples + each - 1) / each;
    return gradient ? round_up((uint64_t)blocks * labels * columns * 4, 256) : 0;
}

int few_labels_loss(const FewLabels &p, float *losses, float *normalisers, cudaStream_t stream)
{
    Args a = {};
    a.p = p, a.losses = losses, a.normalisers_out = normalisers;
    return run<kLoss>(a, stream);
}

int few_labels_predict(const FewLabels &p, int64_t *labels, float *log_probabilities, cudaStream_t stream)
{
    Args a = {};
    a.p = p, a.labels_out = (long long *)labels, a.log_probabilities = log_probabilities;
    return run<kPredict>(a, stream);
}

int few_labels_gradient(const FewLabels &p, const float *normalisers, const float *gradients, int64_t gradients_step, void *dx, void *dw, void *workspace, cudaStream_t stream)
{
    Args a = {};
    a.p = p, a.normalisers = normalisers, a.gradients = gradients, a.gradients_step = (int)gradients_step, a.dx = dx, a.partial = (float *)workspace;
    GTM_TRY(run<kGradient>(a, stream));
    const long long size = p.labels * p.columns;
    const int blocks = (int)((p.examples + a.per_block - 1) / a.per_block);
    const unsigned grid = (unsigned)((size + 31) / 32);
    if (p.type == GTM_F32) return launch_early(few_labels_join_kernel<float>, dim3(grid), dim3(256), 0, stream, a.partial, blocks, size, (float *)dw);
    if (p.type == GTM_BF16) return launch_early(few_labels_join_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, stream, a.partial, blocks, size, (__nv_bfloat16 *)dw);
    return launch_early(few_labels_join_kernel<__half>, dim3(grid), dim3(256), 0, stream, a.partial, blocks, size, (__half *)dw);
}

}  // namespace gtm_readout
