// The softmax operators for a handful of labels (gtm_readout_few_labels.cu), as the entry points in gtm_readout_softmax.cu call them.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gtm_readout {

struct FewLabels {
    int type;
    int64_t examples, labels, columns;
    const void *x, *w;
    int64_t x_stride, w_stride;
    const void *wanted;                 // labels of the examples; null in a prediction
    int wanted_64;
    int64_t ignored;
    float scale;
};

constexpr int64_t kFewLabelsExamples = (int64_t)1 << 16;

// Whether these kernels take a problem, its loss, its gradient and its prediction alike.
bool few_labels(int64_t examples, int64_t labels, int64_t columns);
uint64_t few_labels_workspace(int64_t examples, int64_t labels, int64_t columns, bool gradient);
int few_labels_loss(const FewLabels &p, float *losses, float *normalisers, cudaStream_t stream);
int few_labels_predict(const FewLabels &p, int64_t *labels, float *log_probabilities, cudaStream_t stream);
int few_labels_gradient(const FewLabels &p, const float *normalisers, const float *gradients, int64_t gradients_step, void *dx, void *dw, void *workspace, cudaStream_t stream);

}  // namespace gtm_readout
