// One AdamW step over many tensors.
//
//   g = gradient * gradient_scale      m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g g      u = sqrt(v)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (u / sqrt(1 - b2^t) + eps)
//
// in 32 bits, every operation rounded by itself, p rounded once to its type.  The moments of all tensors lie in two flat
// arrays in which every tensor starts at a multiple of kBlock elements.
//
// 8-bit states: of kBlock elements, m and u are held as e4m3 codes times one 32-bit scale (largest magnitude / 448).  u and not
// v, because a root has half the exponent range of its square.  A code is one of the two neighbours of the value, the upper one with the
// probability of its nearness: an average with b2 = 0.999 moves by 0.1 % a step, less than half the 6 % between neighbours, and
// rounding to nearest would leave it where it is.  The random bits are a hash of (seed, t, element), so a step can be
// repeated.  A u above zero never gets the code of zero, or the next step would divide m by eps alone.
#include "gtm_readout.cuh"

namespace gtm_readout {
namespace {

constexpr int kBlock = 256;                   // elements of a warp's turn, and of one 8-bit scale
constexpr int kTensors = 512;                 // tensors of one launch: their table travels with the launch's arguments
constexpr float kLeastScale = 1.1754943508222875e-38f, kLeastCode = 0.001953125f;

struct AdamTensor {
    void *param;
    const void *gradient;
    void *copy;                               // the parameter once more, in another type; may be null
    long long count, block;                   // first block of the flat arrays
};

struct AdamArgs {
    float b1, other1, b2, other2, decay, eps, gradient_scale;
    double lr, beta1, beta2;
    const long long *steps;                   // steps taken before this one
    void *first, *second;
    float *first_scales, *second_scales;
    unsigned seed;
    int tensors, copy_type;
    long long blocks;                         // of this launch
    AdamTensor t[kTensors];
};
static_assert(sizeof(AdamArgs) <= 32764, "kernel arguments");

// Finaliser of MurmurHash3 (A. Appleby).
__device__ __forceinline__ unsigned mix(unsigned x)
{
    x = (x ^ (x >> 16)) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

__device__ __forceinline__ float root_fast(float v)
{
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Values of four codes.
__device__ __forceinline__ void decode4(unsigned codes, float (&v)[4])
{
    unsigned low, high;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(low) : "h"((unsigned short)codes));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(high) : "h"((unsigned short)(codes >> 16)));
    const float2 a = __half22float2(reinterpret_cast<const __half2 &>(low)), b = __half22float2(reinterpret_cast<const __half2 &>(high));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}

// Codes of four values that are codes' values already (NaN stays NaN).
__device__ __forceinline__ unsigned encode4(const float (&v)[4])
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

template <class T>
__device__ __forceinline__ void load4(const T *p, long long i, long long n, bool wide, float (&v)[4])
{
    if (wide && i + 4 <= n) {
        const Pack<T, 4> q = *(const Pack<T, 4> *)(p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = to_float(q.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = i + k < n ? to_float(p[i + k]) : 0.f;
    }
}

template <class T>
__device__ __forceinline__ void store4(T *p, long long i, long long n, bool wide, const float (&v)[4])
{
    if (wide && i + 4 <= n) {
        Pack<T, 4> q;
#pragma unroll
        for (int k = 0; k < 4; k++) q.v[k] = from_float<T>(v[k]);
        *(Pack<T, 4> *)(p + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i + k < n) p[i + k] = from_float<T>(v[k]);
    }
}

template <class P, class G, bool kNarrow>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamArgs a)
{
    __shared__ float constants[2];
    __shared__ unsigned key_shared;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        const long long step = *a.steps + 1;
        const double t = (double)step;
        constants[0] = (float)(a.lr / (1.0 - pow(a.beta1, t)));
        constants[1] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, t)));
        key_shared = mix(mix(a.seed) + (unsigned)step);
    }
    __syncthreads();
    const float step_size = constants[0], root_correction = constants[1];
    const unsigned key = key_shared;
    int at = 0;
    for (long long b = (long long)blockIdx.x * 8 + threadIdx.x / 32; b < a.blocks; b += (long long)gridDim.x * 8) {
        const long long block = a.t[0].block + b;
        while (at + 1 < a.tensors && a.t[at + 1].block <= block) at++;
        const AdamTensor &t = a.t[at];
        const long long i0 = (block - t.block) * kBlock;           // of the tensor
        const long long n = t.count;
        const bool wide_p = (uintptr_t)t.param % (4 * sizeof(P)) == 0, wide_g = (uintptr_t)t.gradient % (4 * sizeof(G)) == 0;
        float p[2][4], g[2][4], m[2][4], u[2][4];
        unsigned codes_m[2], codes_u[2];
        float scale_m = 0.f, scale_u = 0.f;
        if (kNarrow) scale_m = a.first_scales[block], scale_u = a.second_scales[block];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const long long i = i0 + j * 128 + lane * 4, flat = block * kBlock + j * 128 + lane * 4;
            load4((const P *)t.param, i, n, wide_p, p[j]);
            load4((const G *)t.gradient, i, n, wide_g, g[j]);
            if (kNarrow) {
                codes_m[j] = *(const unsigned *)((const unsigned char *)a.first + flat);
                codes_u[j] = *(const unsigned *)((const unsigned char *)a.second + flat);
            } else {
                load4((const float *)a.first, flat, flat + 4, true, m[j]);
                load4((const float *)a.second, flat, flat + 4, true, u[j]);
            }
        }
        float largest_m = 0.f, largest_u = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (kNarrow) decode4(codes_m[j], m[j]), decode4(codes_u[j], u[j]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float gr = __fmul_rn(g[j][k], a.gradient_scale);
                if (kNarrow) {
                    m[j][k] = __fmul_rn(m[j][k], scale_m);
                    u[j][k] = __fmul_rn(u[j][k], scale_u);
                    u[j][k] = __fmul_rn(u[j][k], u[j][k]);
                }
                m[j][k] = __fadd_rn(__fmul_rn(m[j][k], a.b1), __fmul_rn(gr, a.other1));
                u[j][k] = __fadd_rn(__fmul_rn(u[j][k], a.b2), __fmul_rn(__fmul_rn(gr, gr), a.other2));
                // next to 8-bit states the hardware's root (2^-23) and quotient (2^-22) are exact enough, and a third of the instructions
                const float root = kNarrow ? root_fast(u[j][k]) : __fsqrt_rn(u[j][k]);
                const float below = __fadd_rn(__fmul_rn(root, root_correction), a.eps);
                const float moved = kNarrow ? __fdividef(m[j][k], below) : __fdiv_rn(m[j][k], below);
                p[j][k] = __fsub_rn(__fmul_rn(p[j][k], a.decay), __fmul_rn(step_size, moved));
                if (kNarrow) {
                    u[j][k] = root;
                    largest_m = fmaxf(largest_m, fabsf(m[j][k]));           // NaN is passed over
                    largest_u = fmaxf(largest_u, root);
                }
            }
        }
        if (kNarrow) {
#pragma unroll
            for (int o = 16; o; o /= 2) {
                largest_m = fmaxf(largest_m, __shfl_xor_sync(~0u, largest_m, o));
                largest_u = fmaxf(largest_u, __shfl_xor_sync(~0u, largest_u, o));
            }
            if (!finite(largest_m) || !finite(largest_u)) {
                // infinities are held as NaN and have no part in the scale
                largest_m = largest_u = 0.f;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (finite(m[j][k])) largest_m = fmaxf(largest_m, fabsf(m[j][k]));
                        else m[j][k] = __int_as_float(0x7fffffff);
                        if (finite(u[j][k])) largest_u = fmaxf(largest_u, u[j][k]);
                        else u[j][k] = __int_as_float(0x7fffffff);
                    }
#pragma unroll
                for (int o = 16; o; o /= 2) {
                    largest_m = fmaxf(largest_m, __shfl_xor_sync(~0u, largest_m, o));
                    largest_u = fmaxf(largest_u, __shfl_xor_sync(~0u, largest_u, o));
                }
            }
            scale_m = fmaxf(__fmul_rn(largest_m, (float)(1.0 / 448.0)), kLeastScale);
            scale_u = fmaxf(__fmul_rn(largest_u, (float)(1.0 / 448.0)), kLeastScale);
            const float inverse_m = __fdiv_rn(1.f, scale_m), inverse_u = __fdiv_rn(1.f, scale_u);
            if (lane == 0) a.first_scales[block] = scale_m, a.second_scales[block] = scale_u;
            const unsigned flat = (unsigned)(block * kBlock) + lane * 4;
            bool small = false;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                unsigned random[4];
                float qm[4], qu[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    random[k] = mix((flat + j * 128 + k) * 0x9e3779b1u + key);
                    qm[k] = __fmul_rn(fabsf(m[j][k]), inverse_m), qu[k] = __fmul_rn(u[j][k], inverse_u);
                    small |= !(qm[k] >= 0.015625f) | !(qu[k] >= 0.015625f);
                }
                if (!__any_sync(~0u, small)) {
#pragma unroll
                    for (int k = 0; k < 4; k++) qm[k] = round_normal(qm[k], random[k] >> 16), qu[k] = round_normal(qu[k], random[k] & 0xffff);
                } else {                                             // zeros, NaN, and one in thousands of usual values
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        qm[k] = qm[k] >= 0.015625f ? round_normal(qm[k], random[k] >> 16) : round_small(qm[k], random[k] >> 16);
                        qu[k] = qu[k] >= 0.015625f ? round_normal(qu[k], random[k] & 0xffff) : round_small(qu[k], random[k] & 0xffff);
                        if (u[j][k] > 0.f) qu[k] = fmaxf(qu[k], kLeastCode);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; k++) qm[k] = copysignf(qm[k], m[j][k]);
                codes_m[j] = encode4(qm), codes_u[j] = encode4(qu);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const long long i = i0 + j * 128 + lane * 4, flat = block * kBlock + j * 128 + lane * 4;
            store4((P *)t.param, i, n, wide_p, p[j]);
            if (t.copy) {
                // the copy of the parameter as it is held
#pragma unroll
                for (int k = 0; k < 4; k++) p[j][k] = to_float(from_float<P>(p[j][k]));
                const bool wide_c = (uintptr_t)t.copy % 8 == 0;
                if (a.copy_type == GTM_BF16) store4((__nv_bfloat16 *)t.copy, i, n, wide_c, p[j]);
                else store4((__half *)t.copy, i, n, wide_c, p[j]);
            }
            if (kNarrow) {
                *(unsigned *)((unsigned char *)a.first + flat) = codes_m[j];
                *(unsigned *)((unsigned char *)a.second + flat) = codes_u[j];
            } else {
                store4((float *)a.first, flat, flat + 4, true, m[j]);
                store4((float *)a.second, flat, flat + 4, true, u[j]);
            }
        }
    }
}

__global__ void adamw_count_kernel(long long *steps) { *steps += 1; }

template <class P, class G>
int launch(const AdamArgs &a, bool narrow, cudaStream_t stream)
{
    int device = 0, sms = 0;
    GTM_CU(cudaGetDevice(&device));
    GTM_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    const long long want = (a.blocks + 7) / 8, most = (long long)sms * 8;
    const unsigned grid = (unsigned)(want < most ? want : most);
    if (narrow) adamw_kernel<P, G, true><<<grid, 256, 0, stream>>>(a);
    else adamw_kernel<P, G, false><<<grid, 256, 0, stream>>>(a);
    GTM_CU(cudaGetLastError());
    return GTM_OK;
}

template <class P>
int launch(const AdamArgs &a, int gradient_type, bool narrow, cudaStream_t stream)
{
    return gradient_type == GTM_F32    ? launch<P, float>(a, narrow, stream)
           : gradient_type == GTM_BF16 ? launch<P, __nv_bfloat16>(a, narrow, stream)
                                       : launch<P, __half>(a, narrow, stream);
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
    DeviceGuard guard(device);
    GTM_TRY(guard.status);
    cudaStream_t stream = (cudaStream_t)cuda_stream;
    AdamArgs a;
    a.b1 = (float)beta1, a.other1 = (float)(1 - beta1), a.b2 = (float)beta2, a.other2 = (float)(1 - beta2);
    a.decay = (float)(1 - lr * weight_decay), a.eps = (float)eps, a.gradient_scale = (float)gradient_scale;
    a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.steps = (const long long *)steps, a.seed = seed;
    a.first = first, a.second = second, a.first_scales = first_scales, a.second_scales = second_scales, a.copy_type = copy_type;
    long long block = 0;
    for (int64_t i = 0; i < number_of_tensors;) {
        a.tensors = 0, a.blocks = 0;
        for (; i < number_of_tensors && a.tensors < kTensors; i++) {
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
    adamw_count_kernel<<<1, 1, 0, stream>>>((long long *)steps);
    GTM_CU(cudaGetLastError());
    return GTM_OK;
}
