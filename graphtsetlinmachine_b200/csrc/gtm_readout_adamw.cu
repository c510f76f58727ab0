// One AdamW step over many tensors.
//
//   g = gradient * gradient_scale      m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g g      u = sqrt(v)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (u / sqrt(1 - b2^t) + eps)
//
// in 32 bits, p rounded once to its type.  The moments of all tensors lie in two flat
// arrays in which every tensor starts at a multiple of kBlock elements.
//
// 8-bit states: of kBlock elements, m and u are held as e4m3 codes times one 32-bit scale (largest magnitude / 448).  u and not
// v, because a root has half the exponent range of its square.  A code is one of the two neighbours of the value, the upper one with the
// probability of its nearness: an average with b2 = 0.999 moves by 0.1 % a step, less than half the 6 % between neighbours, and
// rounding to nearest would leave it where it is.  The random bits are a hash of (seed, t, element), so a step can be
// repeated.  A u above zero never gets the code of zero, or the next step would divide m by eps alone.
#include "gtm_readout.cuh"

#include <algorithm>
#include <memory>
#include <new>

namespace gtm_readout {
namespace {

// What bounds a step in 32 bits is memory: 60 M fp32 parameters with bf16 gradients take 258 us, 6.0 TB/s of 26 bytes each.
constexpr int kBlock = 256;                   // elements of a warp's turn, and of one 8-bit scale
constexpr int kTensors = 512, kFewTensors = 16;  // tensors of one launch, whose table travels with its arguments: a long one (20 KB) or a short one
constexpr float kLeastScale = 1.1754943508222875e-38f, kLeastCode = 0.001953125f;

struct AdamTensor {
    void *param;
    const void *gradient;
    void *copy;                               // the parameter once more, in another type; may be null
    long long count, block;                   // first block of the flat arrays
};

struct AdamHead {
    float b1, other1, b2, other2, decay, eps, gradient_scale;
    double lr, beta1, beta2;
    const long long *steps;                   // steps taken before this one
    void *first, *second;
    float *first_scales, *second_scales;
    unsigned seed;
    int tensors, copy_type;
    long long blocks;                         // of this launch
};

template <int kMost>
struct AdamArgs : AdamHead {
    AdamTensor t[kMost];
};
static_assert(sizeof(AdamArgs<kTensors>) <= 32764, "kernel arguments");

// Finaliser of MurmurHash3 (A. Appleby).
__device__ __forceinline__ unsigned mix(unsigned x)
{
    x = (x ^ (x >> 16)) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

__device__ __forceinline__ float reciprocal_fast(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Values of four codes.
__device__ __forceinline__ void decode4(unsigned codes, float *v)
{
    unsigned low, high;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(low) : "h"((unsigned short)codes));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(high) : "h"((unsigned short)(codes >> 16)));
    const float2 a = __half22float2(reinterpret_cast<const __half2 &>(low)), b = __half22float2(reinterpret_cast<const __half2 &>(high));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

// Codes of four values that are codes' values already (NaN stays NaN).
__device__ __forceinline__ unsigned encode4(const float *v)
{
    unsigned short low, high;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(v[1]), "f"(v[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(v[3]), "f"(v[2]));
    return low | (unsigned)high << 16;
}

// The code's value that a magnitude in units of the scale is rounded to, with 16 random bits.  Normal values (2^-6 and above) have four
// bits of fraction: random bits are added below and what is below is cut off.  Smaller ones are multiples of 2^-9.
__device__ __forceinline__ float round_normal(float r, unsigned random) { return __uint_as_float((__float_as_uint(r) + (random << 4)) & ~0xfffffu); }
__device__ __forceinline__ float round_small(float r, unsigned random)
{
    const float below_one = __uint_as_float(0x3f800000u | random << 7) - 1.f;      // random / 2^16
    return floorf(__fadd_rn(__fmul_rn(r, 512.f), below_one)) * kLeastCode;
}

// A lane's elements in a row: all of them, at a boundary of the load (or store), or element by element as far as the tensor goes (zeros behind it).
template <class T, int N>
__device__ __forceinline__ void load_some(const T *p, long long i, long long n, Pack<T, N> &v)
{
#pragma unroll
    for (int k = 0; k < N; k++) v.v[k] = i + k < n ? p[i + k] : from_float<T>(0.f);
}

template <class T, int N>
__device__ __forceinline__ void load_all(const T *p, long long i, Pack<T, N> &v)
{
    constexpr int kWide = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
    for (int k = 0; k < N; k += kWide) reinterpret_cast<Pack<T, kWide> &>(v.v[k]) = *(const Pack<T, kWide> *)(p + i + k);
}

template <class T, int N>
__device__ __forceinline__ void store(T *p, long long i, long long n, bool whole, const float (&v)[N])
{
    constexpr int kWide = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
    Pack<T, N> q;
#pragma unroll
    for (int k = 0; k < N; k++) q.v[k] = from_float<T>(v[k]);
    if (whole) {
#pragma unroll
        for (int k = 0; k < N; k += kWide) *(Pack<T, kWide> *)(p + i + k) = reinterpret_cast<const Pack<T, kWide> &>(q.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (i + k < n) p[i + k] = q.v[k];
    }
}

// What hangs on the number of the step, once per block.
struct StepConstants {
    float step_size, root_correction;
    unsigned key;
};

__device__ __forceinline__ StepConstants step_constants(const AdamHead &a)
{
    __shared__ StepConstants c;
    if (threadIdx.x == 0) {
        const long long step = *a.steps + 1;
        const double t = (double)step;
        c.step_size = (float)(a.lr / (1.0 - pow(a.beta1, t)));
        c.root_correction = (float)(1.0 / sqrt(1.0 - pow(a.beta2, t)));
        c.key = mix(mix(a.seed) + (unsigned)step);
    }
    __syncthreads();
    return c;
}

// Whether a block of a tensor is there as a whole, at boundaries of 16 bytes.
template <class P, class G>
__device__ __forceinline__ bool is_whole(const AdamTensor &t, long long i)
{
    return (((uintptr_t)t.param | (uintptr_t)t.gradient | (uintptr_t)t.copy) & 15) == 0 && i / kBlock * kBlock + kBlock <= t.count;
}

// The parameter as it is held, and its copy.
template <class P, int N>
__device__ __forceinline__ void store_param(const AdamHead &a, const AdamTensor &t, long long i, bool whole, float (&p)[N])
{
    store((P *)t.param, i, t.count, whole, p);
    if (!t.copy) return;
#pragma unroll
    for (int k = 0; k < N; k++) p[k] = to_float(from_float<P>(p[k]));
    if (a.copy_type == GTM_BF16) store((__nv_bfloat16 *)t.copy, i, t.count, whole, p);
    else store((__half *)t.copy, i, t.count, whole, p);
}

template <class P, class G, int kMost>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamArgs<kMost> a)
{
    next_may_start();
    wait_for_previous();
    const int lane = threadIdx.x & 31;
    const StepConstants c = step_constants(a);
    int at = 0;
    for (long long b = (long long)blockIdx.x * 8 + threadIdx.x / 32; b < a.blocks; b += (long long)gridDim.x * 8) {
        const long long block = a.t[0].block + b;
        while (at + 1 < a.tensors && a.t[at + 1].block <= block) at++;
        const AdamTensor &t = a.t[at];
        // four elements, and four 128 further: 16 bytes of 32-bit arrays, one next to the other over the warp
        const long long flat = block * kBlock + lane * 4, i = flat - t.block * kBlock;
        const bool whole = is_whole<P, G>(t, i);
        Pack<P, 4> p4[2];
        Pack<G, 4> g4[2];
        Pack<float, 4> m[2], v[2];
#pragma unroll
        for (int j = 0; j < 2; j++) m[j] = *(const Pack<float, 4> *)((const float *)a.first + flat + j * 128), v[j] = *(const Pack<float, 4> *)((const float *)a.second + flat + j * 128);
        if (whole) {
#pragma unroll
            for (int j = 0; j < 2; j++) p4[j] = *(const Pack<P, 4> *)((const P *)t.param + i + j * 128), g4[j] = *(const Pack<G, 4> *)((const G *)t.gradient + i + j * 128);
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) load_some((const P *)t.param, i + j * 128, t.count, p4[j]), load_some((const G *)t.gradient, i + j * 128, t.count, g4[j]);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float p[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float g = __fmul_rn(to_float(g4[j].v[k]), a.gradient_scale);
                m[j].v[k] = __fadd_rn(__fmul_rn(m[j].v[k], a.b1), __fmul_rn(g, a.other1));
                v[j].v[k] = __fadd_rn(__fmul_rn(v[j].v[k], a.b2), __fmul_rn(__fmul_rn(g, g), a.other2));
                const float moved = __fdiv_rn(m[j].v[k], __fadd_rn(__fmul_rn(__fsqrt_rn(v[j].v[k]), c.root_correction), a.eps));
                p[k] = __fsub_rn(__fmul_rn(to_float(p4[j].v[k]), a.decay), __fmul_rn(c.step_size, moved));
            }
            *(Pack<float, 4> *)((float *)a.first + flat + j * 128) = m[j];
            *(Pack<float, 4> *)((float *)a.second + flat + j * 128) = v[j];
            store_param<P>(a, t, i + j * 128, whole, p);
        }
    }
}

// States of 8 bits.  The moments are computed operation by operation as in 32 bits: a last bit can decide between two codes, and with it what the states
// are from then on.  The parameter is not among them: its quotient is the hardware's reciprocal (2^-23) in fused operations.  What bounds it is
// instructions, 85 an element, the root, the hash and the roundings being half of them: 592 us for 200 M bf16 parameters (3.4 TB/s).  Loading the next block
// before the present one is worked on took 1,130 us: two registers for every one loaded left half as many warps.
template <class P, class G, int kMost>
__global__ void __launch_bounds__(256, 4) adamw_narrow_kernel(const __grid_constant__ AdamArgs<kMost> a)
{
    next_may_start();
    wait_for_previous();
    const int lane = threadIdx.x & 31;
    const StepConstants c = step_constants(a);
    int at = 0;
    for (long long b = (long long)blockIdx.x * 8 + threadIdx.x / 32; b < a.blocks; b += (long long)gridDim.x * 8) {
        const long long block = a.t[0].block + b;
        while (at + 1 < a.tensors && a.t[at + 1].block <= block) at++;
        const AdamTensor &t = a.t[at];
        const long long flat = block * kBlock + lane * 8, i = flat - t.block * kBlock;
        const bool whole = is_whole<P, G>(t, i);
        const uint2 codes_m = *(const uint2 *)((const unsigned char *)a.first + flat), codes_u = *(const uint2 *)((const unsigned char *)a.second + flat);
        const float held_m = a.first_scales[block], held_u = a.second_scales[block];
        Pack<P, 8> p8;
        Pack<G, 8> g8;
        if (whole) load_all((const P *)t.param, i, p8), load_all((const G *)t.gradient, i, g8);      // the warp is of one mind: no load waits for another
        else load_some((const P *)t.param, i, t.count, p8), load_some((const G *)t.gradient, i, t.count, g8);
        float p[8], m[8], u[8];
        decode4(codes_m.x, m), decode4(codes_m.y, m + 4), decode4(codes_u.x, u), decode4(codes_u.y, u + 4);
        float largest_m = 0.f, largest_u = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float g = __fmul_rn(to_float(g8.v[k]), a.gradient_scale);
            m[k] = __fadd_rn(__fmul_rn(__fmul_rn(m[k], held_m), a.b1), __fmul_rn(g, a.other1));
            u[k] = __fmul_rn(u[k], held_u);
            u[k] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(u[k], u[k]), a.b2), __fmul_rn(__fmul_rn(g, g), a.other2)));
            const float moved = m[k] * reciprocal_fast(fmaf(u[k], c.root_correction, a.eps));
            p[k] = fmaf(-c.step_size, moved, to_float(p8.v[k]) * a.decay);
            largest_m = fmaxf(largest_m, fabsf(m[k]));               // NaN is passed over
            largest_u = fmaxf(largest_u, u[k]);
        }
        store_param<P>(a, t, i, whole, p);
        // magnitudes: their bits have their order
        largest_m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(largest_m)));
        largest_u = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(largest_u)));
        if (!finite(largest_m) || !finite(largest_u)) {
            // infinities are held as NaN and have no part in the scale
            largest_m = largest_u = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (finite(m[k])) largest_m = fmaxf(largest_m, fabsf(m[k]));
                else m[k] = __int_as_float(0x7fffffff);
                if (finite(u[k])) largest_u = fmaxf(largest_u, u[k]);
                else u[k] = __int_as_float(0x7fffffff);
            }
            largest_m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(largest_m)));
            largest_u = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(largest_u)));
        }
        const float scale_m = fmaxf(largest_m * (float)(1.0 / 448.0), kLeastScale), scale_u = fmaxf(largest_u * (float)(1.0 / 448.0), kLeastScale);
        const float inverse_m = __fdiv_rn(1.f, scale_m), inverse_u = __fdiv_rn(1.f, scale_u);
        if (lane == 0) a.first_scales[block] = scale_m, a.second_scales[block] = scale_u;
        unsigned random[8];
        float qm[8], qu[8];
        bool normal = true;
        const unsigned from = (unsigned)flat * 0x9e3779b1u + c.key;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            random[k] = mix(from + k * 0x9e3779b1u);
            qm[k] = fabsf(m[k]) * inverse_m, qu[k] = u[k] * inverse_u;
            normal &= qm[k] >= 0.015625f && qu[k] >= 0.015625f;          // not for NaN
        }
        if (__all_sync(~0u, normal)) {
#pragma unroll
            for (int k = 0; k < 8; k++) qm[k] = round_normal(qm[k], random[k] >> 16), qu[k] = round_normal(qu[k], random[k] & 0xffff);
        } else {                                                  // zeros, NaN, and one in thousands of usual values
#pragma unroll
            for (int k = 0; k < 8; k++) {
                qm[k] = qm[k] >= 0.015625f ? round_normal(qm[k], random[k] >> 16) : round_small(qm[k], random[k] >> 16);
                qu[k] = qu[k] >= 0.015625f ? round_normal(qu[k], random[k] & 0xffff) : round_small(qu[k], random[k] & 0xffff);
                if (u[k] > 0.f) qu[k] = fmaxf(qu[k], kLeastCode);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; k++) qm[k] = copysignf(qm[k], m[k]);
        *(uint2 *)((unsigned char *)a.first + flat) = make_uint2(encode4(qm), encode4(qm + 4));
        *(uint2 *)((unsigned char *)a.second + flat) = make_uint2(encode4(qu), encode4(qu + 4));
    }
}

__global__ void adamw_count_kernel(long long *steps)
{
    next_may_start();
    wait_for_previous();
    *steps += 1;
}

template <class P, class G, int kMost>
int launch(const AdamArgs<kMost> &a, bool narrow, cudaStream_t stream)
{
    int device = 0, sms = 0;
    GTM_CU(cudaGetDevice(&device));
    GTM_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    const long long want = (a.blocks + 7) / 8, most = (long long)sms * 8;
    const unsigned grid = (unsigned)(want < most ? want : most);
    return launch_early(narrow ? adamw_narrow_kernel<P, G, kMost> : adamw_kernel<P, G, kMost>, dim3(grid), dim3(256), 0, stream, a);
}

template <class P, int kMost>
int launch(const AdamArgs<kMost> &a, int gradient_type, bool narrow, cudaStream_t stream)
{
    return gradient_type == GTM_F32    ? launch<P, float>(a, narrow, stream)
           : gradient_type == GTM_BF16 ? launch<P, __nv_bfloat16>(a, narrow, stream)
                                       : launch<P, __half>(a, narrow, stream);
}

// All tensors of a step, kMost of them at a time.
template <int kMost>
int launch_all(const AdamHead &head, int64_t number_of_tensors, const int64_t *counts, int param_type, const void *const *params, int gradient_type, const void *const *gradients,
               const void *const *copies, bool narrow, cudaStream_t stream)
{
    AdamArgs<kMost> a;
    static_cast<AdamHead &>(a) = head;
    long long block = 0;
    for (int64_t i = 0; i < number_of_tensors;) {
        a.tensors = 0, a.blocks = 0;
        for (; i < number_of_tensors && a.tensors < kMost; i++) {
            if (counts[i] == 0) continue;
            a.t[a.tensors++] = {(void *)params[i], gradients[i], copies ? (void *)copies[i] : nullptr, counts[i], block};
            const long long blocks = (counts[i] + kBlock - 1) / kBlock;
            block += blocks, a.blocks += blocks;
        }
        if (a.tensors == 0) break;
        GTM_TRY(param_type == GTM_F32    ? launch<float>(a, gradient_type, narrow, stream)
                : param_type == GTM_BF16 ? launch<__nv_bfloat16>(a, gradient_type, narrow, stream)
                                         : launch<__half>(a, gradient_type, narrow, stream));
    }
    return GTM_OK;
}

// Memory that a step touches.
struct Range {
    uintptr_t first, end;
    bool written;
};

// Whether something written meets anything else: the order of two writes, or of a read and a write, would be open.  Gradients may share memory.
bool overlap(Range *ranges, size_t count)
{
    std::sort(ranges, ranges + count, [](const Range &a, const Range &b) { return a.first < b.first; });
    uintptr_t written = 0, any = 0;               // ends so far
    for (size_t i = 0; i < count; i++) {
        if (ranges[i].first < (ranges[i].written ? any : written)) return true;
        any = std::max(any, ranges[i].end);
        if (ranges[i].written) written = std::max(written, ranges[i].end);
    }
    return false;
}

}  // namespace
}  // namespace gtm_readout

using namespace gtm_readout;

extern "C" int gtm_adamw_step(int device, void *cuda_stream, int64_t number_of_tensors, const int64_t *counts, int param_type, const void *const *params,
                              int gradient_type, const void *const *gradients, int copy_type, const void *const *copies, int state_bits, void *first,
                              void *second, float *first_scales, float *second_scales, int64_t *steps, double lr, double beta1, double beta2, double eps,
                              double weight_decay, double gradient_scale, uint32_t seed)
{
    if (number_of_tensors < 0 || (number_of_tensors && (!counts || !params || !gradients))) return fail(GTM_ERR_ARG, "gtm_adamw_step: null list of tensors");
    if (!type_bytes(param_type) || !type_bytes(gradient_type)) return fail(GTM_ERR_ARG, "gtm_adamw_step: element type %d or %d is none of GTM_F32, GTM_BF16, GTM_F16", param_type, gradient_type);
    if (copies && copy_type != GTM_BF16 && copy_type != GTM_F16) return fail(GTM_ERR_ARG, "gtm_adamw_step: copies are GTM_BF16 or GTM_F16");
    if (state_bits != 8 && state_bits != 32) return fail(GTM_ERR_ARG, "gtm_adamw_step: states of %d bits (8 or 32)", state_bits);
    if (!steps || (uintptr_t)steps % 8) return fail(GTM_ERR_ARG, "gtm_adamw_step: null or misaligned step count");
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) return fail(GTM_ERR_ARG, "gtm_adamw_step: betas %g and %g are not in [0, 1)", beta1, beta2);
    if (!(eps >= 0) || !(lr >= 0) || !(weight_decay >= 0)) return fail(GTM_ERR_ARG, "gtm_adamw_step: negative lr, eps or weight decay");
    const bool narrow = state_bits == 8;
    int64_t all = 0;
    for (int64_t i = 0; i < number_of_tensors; i++) {
        if (counts[i] < 0) return fail(GTM_ERR_ARG, "gtm_adamw_step: tensor %lld has %lld elements", (long long)i, (long long)counts[i]);
        if (counts[i] == 0) continue;
        if (!params[i] || !gradients[i] || (copies && !copies[i])) return fail(GTM_ERR_ARG, "gtm_adamw_step: tensor %lld is null", (long long)i);
        if ((uintptr_t)params[i] % type_bytes(param_type) || (uintptr_t)gradients[i] % type_bytes(gradient_type) || (copies && (uintptr_t)copies[i] % 2))
            return fail(GTM_ERR_ARG, "gtm_adamw_step: tensor %lld is misaligned", (long long)i);
        all += counts[i];
    }
    if (all && (!first || !second || (uintptr_t)first % 16 || (uintptr_t)second % 16)) return fail(GTM_ERR_ARG, "gtm_adamw_step: null or misaligned states");
    if (all && narrow && (!first_scales || !second_scales)) return fail(GTM_ERR_ARG, "gtm_adamw_step: 8-bit states need scales");
    std::unique_ptr<Range[]> ranges(new (std::nothrow) Range[(size_t)number_of_tensors * 3 + 5]);
    if (!ranges) return fail(GTM_ERR_OOM, "gtm_adamw_step: no memory for a list of %lld tensors", (long long)number_of_tensors);
    size_t count = 0;
    const auto take = [&](const void *p, uint64_t bytes, bool written) {
        if (bytes) ranges[count++] = {(uintptr_t)p, (uintptr_t)p + bytes, written};
    };
    uint64_t blocks = 0;
    for (int64_t i = 0; i < number_of_tensors; i++) {
        take(params[i], counts[i] * type_bytes(param_type), true), take(gradients[i], counts[i] * type_bytes(gradient_type), false);
        if (copies) take(copies[i], counts[i] * 2, true);
        blocks += (counts[i] + kBlock - 1) / kBlock;
    }
    take(steps, 8, true), take(first, blocks * kBlock * (narrow ? 1 : 4), true), take(second, blocks * kBlock * (narrow ? 1 : 4), true);
    if (narrow) take(first_scales, blocks * 4, true), take(second_scales, blocks * 4, true);
    if (overlap(ranges.get(), count)) return fail(GTM_ERR_ARG, "gtm_adamw_step: a tensor, a state or a copy overlaps another");
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    AdamHead a = {};
    a.b1 = (float)beta1, a.other1 = (float)(1 - beta1), a.b2 = (float)beta2, a.other2 = (float)(1 - beta2);
    a.decay = (float)(1 - lr * weight_decay), a.eps = (float)eps, a.gradient_scale = (float)gradient_scale;
    a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.steps = (const long long *)steps, a.seed = seed;
    a.first = first, a.second = second, a.first_scales = first_scales, a.second_scales = second_scales, a.copy_type = copy_type;
    GTM_TRY(number_of_tensors <= kFewTensors ? launch_all<kFewTensors>(a, number_of_tensors, counts, param_type, params, gradient_type, gradients, copies, narrow, stream)
                                             : launch_all<kTensors>(a, number_of_tensors, counts, param_type, params, gradient_type, gradients, copies, narrow, stream));
    return launch_early(adamw_count_kernel, dim3(1), dim3(1), 0, stream, (long long *)steps);
}
