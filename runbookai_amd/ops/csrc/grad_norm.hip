// The norm of many gradients together, and clipping by it (gfx950).
//
//   norm = sqrt(sum over all tensors of g^2),  g *= min(1, limit / (norm + eps))
//
// Bound by memory: the first kernel reads every gradient once, the second reads
// and writes them, or ends at once where the norm is within the limit (decided
// on the device: nothing waits for the host).  The tensors' addresses travel as
// kernel arguments, up to 128 a launch, so there is no table to copy and a
// captured graph keeps its own.
//
// A workgroup takes chunks of 8192 elements, at most 1024 workgroups a launch (4 a
// CU): enough loads on their way, and few partial sums for the second kernel to
// add.  1.75 GB of bf16: sums 0.33 ms (5.2 TB/s), clipping 0.68 ms (5.1 TB/s);
// 88 MB of fp32: 15 us (5.8 TB/s, partly cached) and 31 us; 13 MB within the
// limit: 4.9 and 2.9 us.
//
// The squares are summed in fp64, which costs nothing beside the reads: no
// gradient's square leaves the range (fp32's ends at |g| = 1.8e19), and tiny
// ones stay in.  The factor is fp64 too (1e-3 / 1e38 is no normal fp32 number).
// Every workgroup writes one partial sum; in the second kernel every workgroup adds
// all of them in the same order, so all have the same factor and the same gradients
// give the same bits.
#include "common.h"

#include "grad_norm.h"

namespace {

template <typename T> using Vec16 = T __attribute__((ext_vector_type(16 / sizeof(T))));

// The chunks of a launch that are this workgroup's: f(tensor, first element).
// Elements are counted from the 16-byte boundary at or before the tensor's
// start, so that a chunk's vectors are aligned wherever a tensor begins.
template <typename F>
DEVINL void each_chunk(const GradTable& t, F f) {
    const int all = t.first[t.n];
    for (int c = blockIdx.x; c < all; c += gridDim.x) {
        int lo = 0, hi = t.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (t.first[mid] <= c) lo = mid;
            else hi = mid - 1;
        }
        f(lo, (long)(c - t.first[lo]) * GRAD_CHUNK);
    }
}

template <typename T>
DEVINL double chunk_sum(const void* p, long n, long at) {
    constexpr int VEC = 16 / sizeof(T), PER = GRAD_CHUNK / VEC / 256;
    const unsigned long a = reinterpret_cast<unsigned long>(p);
    const long skip = (long)(a & 15) / (long)sizeof(T);
    const T* base = reinterpret_cast<const T*>(a & ~15ul);
    const long end = skip + n;
    Vec16<T> v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long e = at + (long)(threadIdx.x + i * 256) * VEC;
        v[i] = Vec16<T>{};
        if (e >= skip && e + VEC <= end) {
            v[i] = *reinterpret_cast<const Vec16<T>*>(base + e);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (e + j >= skip && e + j < end) v[i][j] = base[e + j];
        }
    }
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const double g = (double)(float)v[i][j];
            s = fma(g, g, s);
        }
    return s;
}

template <typename T>
DEVINL void chunk_scale(void* p, long n, long at, double f) {
    constexpr int VEC = 16 / sizeof(T), PER = GRAD_CHUNK / VEC / 256;
    const unsigned long a = reinterpret_cast<unsigned long>(p);
    const long skip = (long)(a & 15) / (long)sizeof(T);
    T* base = reinterpret_cast<T*>(a & ~15ul);
    const long end = skip + n;
    Vec16<T> v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long e = at + (long)(threadIdx.x + i * 256) * VEC;
        if (e >= skip && e + VEC <= end) v[i] = *reinterpret_cast<const Vec16<T>*>(base + e);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long e = at + (long)(threadIdx.x + i * 256) * VEC;
        if (e >= skip && e + VEC <= end) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = (T)(float)((double)(float)v[i][j] * f);
            *reinterpret_cast<Vec16<T>*>(base + e) = v[i];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (e + j >= skip && e + j < end) base[e + j] = (T)(float)((double)(float)base[e + j] * f);
        }
    }
}

DEVINL double block_sum(double s) {
    __shared__ double part[4];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, WAVE);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

}  // namespace

__global__ void __launch_bounds__(256)
grad_sums_kernel(GradTable t, double* __restrict__ sums) {
    double s = 0.0;
    each_chunk(t, [&](int i, long at) {
        if (t.kind[i] == 0) s += chunk_sum<float>(t.ptr[i], t.size[i], at);
        else if (t.kind[i] == 1) s += chunk_sum<__bf16>(t.ptr[i], t.size[i], at);
        else s += chunk_sum<_Float16>(t.ptr[i], t.size[i], at);
    });
    s = block_sum(s);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

DEVINL double norm_of(const double* __restrict__ sums, int n) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += sums[i];
    return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(256)
grad_norm_kernel(const double* __restrict__ sums, int n, float* __restrict__ norm) {
    const double x = norm_of(sums, n);
    if (threadIdx.x == 0) *norm = (float)x;
}

__global__ void __launch_bounds__(256)
grad_clip_kernel(GradTable t, const double* __restrict__ sums, int n, double limit, double eps,
                 float* __restrict__ norm) {
    const double x = norm_of(sums, n);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)x;
    const double f = limit / (x + eps);
    if (f >= 1.0) return;   // not for a NaN, which goes into every gradient
    each_chunk(t, [&](int i, long at) {
        if (t.kind[i] == 0) chunk_scale<float>(t.ptr[i], t.size[i], at, f);
        else if (t.kind[i] == 1) chunk_scale<__bf16>(t.ptr[i], t.size[i], at, f);
        else chunk_scale<_Float16>(t.ptr[i], t.size[i], at, f);
    });
}

// ---------------------------------------------------------------- launchers
// Each returns the launch's hipError_t.

extern "C" int launch_grad_sums(const GradTable* t, int blocks, void* sums, void* stream) {
    hipLaunchKernelGGL(grad_sums_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, *t,
                       (double*)sums);
    return (int)hipGetLastError();
}

extern "C" int launch_grad_norm(const void* sums, int n, void* norm, void* stream) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream,
                       (const double*)sums, n, (float*)norm);
    return (int)hipGetLastError();
}

extern "C" int launch_grad_clip(const GradTable* t, int blocks, const void* sums, int n,
                                double limit, double eps, void* norm, void* stream) {
    hipLaunchKernelGGL(grad_clip_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, *t,
                       (const double*)sums, n, limit, eps, (float*)norm);
    return (int)hipGetLastError();
}
