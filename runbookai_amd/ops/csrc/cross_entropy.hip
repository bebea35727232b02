// Cross-entropy of next tokens and its gradient (gfx950).
//
//   loss_i = log sum_j exp(x_ij) - x_it      rows with a label t
//   dx_ij  = (exp(x_ij - m_i) / l_i - [j = t]) g_i
// with m_i the row's maximum and l_i = sum_j exp(x_ij - m_i).
//
// Both kernels are bound by memory.  The forward one reads a labelled row once
// (running maximum and sum in each thread, joined at the end) and keeps m and l
// for the backward one, which reads the row again and writes the gradient; a
// row without a label is not read, and its gradient is written as zeros.  The
// gradient is not made in the forward pass: the factor g that comes back
// (a loss scale, say) has to be in it before it is rounded to 16 bits, where a
// mean's 1/n alone would push small values below fp16's range.
//
// 4096 x 128256 bf16: forward 0.20 ms (5.2 TB/s), gradient 0.37 ms (5.7 TB/s);
// 32768 x 4096 with three of ten rows labelled: 19.5 us (the labelled rows' 81 MB
// at 4.1 TB/s) and 52 us (81 MB read, 268 written: 6.7 TB/s, as the rows were in
// cache).  Where rows have no labels the gradient's zeros are most of the work.
//
// m and l are kept apart, not as one log-sum: x - m is nearly exact, while a
// log-sum near 12 is rounded by 5e-7, which would be in every gradient.
#include "common.h"

#include <type_traits>

// The longest row that a single wave takes; 16 take longer ones.  A step of 16 waves
// is 64 KB of a row, which short rows leave mostly empty; one wave alone is slow where
// the rows are few.  Loss / loss and gradient (us), one wave and 16, bf16 and fp32:
//   65536 x 4096    97/314   458/982    188/607   445/902
//   32768 x 8192    98/316   250/562    190/607   262/596
//   16384 x 16384  100/314   147/351    196/626   176/588
//   8388 x 32000   105/342   102/289    196/654   175/586
//   2092 x 128256  106/388    96/316    206/724   183/622
//   64 x 128256     35/ 93    12/ 61     56/149    13/ 61  (61 is the call's host time)
// So fp32 changes sides here; 16 bits, with twice the columns in a step, would later.
#define XENT_SHORT 8192

namespace {

template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int VEC = 4;
    static DEVINL float get(float v) { return v; }
    static DEVINL float put(float v) { return v; }
};
template <> struct Elem<__bf16> {
    static constexpr int VEC = 8;
    static DEVINL float get(__bf16 v) { return (float)v; }
    static DEVINL __bf16 put(float v) { return (__bf16)v; }
};
template <> struct Elem<_Float16> {
    static constexpr int VEC = 8;
    static DEVINL float get(_Float16 v) { return (float)v; }
    static DEVINL _Float16 put(float v) { return (_Float16)v; }
};
template <typename T>
using Vec = T __attribute__((ext_vector_type(Elem<T>::VEC)));
// the same at any element: one load on this hardware too
template <typename T>
using Loose = T __attribute__((ext_vector_type(Elem<T>::VEC), aligned(sizeof(T))));

constexpr float L2E = 1.4426950408889634f;
constexpr float L2E_LO = 1.9259629911266175e-8f;   // log2(e) - L2E
constexpr float LN2 = 0.6931471805599453f;

// exp(t), t <= 0.  For 32-bit results the product t log2(e) is carried in two
// parts: rounded to one, it alone is off by 6e-8 |t|.
template <typename T>
DEVINL float exp_neg(float t) {
    const float a = t * L2E;
    const float e = __builtin_amdgcn_exp2f(a);
    if (sizeof(T) < 4 || a < -126.f) return e;
    const float rest = fmaf(t, L2E, -a) + t * L2E_LO;
    return fmaf(e, rest * LN2, e);
}

// (m, l) of two parts of a row; a part without a finite value has m = -inf
DEVINL void join(float& m, float& l, float m2, float l2) {
    const float to = fmaxf(m, m2);
    const float base = to == -INFINITY ? 0.f : to;
    l = l * __builtin_amdgcn_exp2f((m - base) * L2E) +
        l2 * __builtin_amdgcn_exp2f((m2 - base) * L2E);
    m = to;
}

// Elements before the row's first 16-byte boundary
template <typename T>
DEVINL int head_of(const T* row, int V) {
    const int h = (int)((16 - (reinterpret_cast<unsigned long>(row) & 15)) & 15) / (int)sizeof(T);
    return min(h, V);
}

}  // namespace

// WAVES waves a row, 4 waves a workgroup at least.  A wave a row needs no
// barrier and reads a row of 4096 in two steps; long rows take 16 (4 a row read
// 128256 bf16 at 5.0 TB/s, 16 at 5.4).  A workgroup leaves one sum and count of
// its rows (`sums` not null) to add up.
template <typename T, int WAVES>
__global__ void __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64)
xent_fwd_kernel(const T* __restrict__ x, long stride, const long* __restrict__ targets,
                long ignore, int N, int V, float* __restrict__ loss,
                float2_t* __restrict__ stats, double* __restrict__ sums,
                int* __restrict__ counts) {
    constexpr int VEC = Elem<T>::VEC, LANES = WAVES * 64;
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    constexpr int U = 4;
    const int tid = threadIdx.x % LANES;
    const long part = (long)blockIdx.y * gridDim.x + blockIdx.x;
    const long row = part * ROWS + threadIdx.x / LANES;
    const long t = row < N ? targets[row] : ignore;
    double sum = 0.0;   // of a row's first thread
    int labels = 0;
    if (row < N && t == ignore && tid == 0) loss[row] = 0.f;
    if (row < N && t != ignore) {   // the whole workgroup, where it has a barrier
        const T* r = x + row * stride;
        float m = -INFINITY, l = 0.f;
        auto one = [&](float v) {
            if (v > m) {
                l *= __builtin_amdgcn_exp2f((m - v) * L2E);
                m = v;
            }
            l += __builtin_amdgcn_exp2f((v - (m == -INFINITY ? 0.f : m)) * L2E);
        };
        const int head = head_of(r, V);
        const int vecs = (V - head) / VEC;
        const Vec<T>* body = reinterpret_cast<const Vec<T>*>(r + head);
        // U vectors on their way at a time, all of them real but in the last step
        auto step = [&](int i0, auto whole) {
            Vec<T> v[U];
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u] = body[whole ? i0 + u * LANES : min(i0 + u * LANES, vecs - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (whole || i0 + u * LANES < vecs)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) top = fmaxf(top, Elem<T>::get(v[u][j]));
            if (top > m) {
                l *= __builtin_amdgcn_exp2f((m - top) * L2E);
                m = top;
            }
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (whole || i0 + u * LANES < vecs)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        l += __builtin_amdgcn_exp2f((Elem<T>::get(v[u][j]) - base) * L2E);
        };
        int i0 = 0;
        for (; i0 + U * LANES <= vecs; i0 += U * LANES) step(i0 + tid, std::true_type{});
        if (i0 < vecs) step(i0 + tid, std::false_type{});
        // the rest: fewer than VEC elements at each end
        const int tail = head + vecs * VEC;
        if (tid < head) one(Elem<T>::get(r[tid]));
        if (tail + tid < V) one(Elem<T>::get(r[tail + tid]));
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const float m2 = __shfl_xor(m, off, WAVE), l2 = __shfl_xor(l, off, WAVE);
            join(m, l, m2, l2);
        }
        if (WAVES > 1) {
            __shared__ float ms[WAVES], lsum[WAVES];
            if ((tid & 63) == 0) { ms[tid >> 6] = m; lsum[tid >> 6] = l; }
            __syncthreads();
            m = ms[0];
            l = lsum[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) join(m, l, ms[w], lsum[w]);
        }
        if (tid == 0) {
            // a label that is no place of the row: no value, and no read
            const bool in = t >= 0 && t < V;
            const float x = in ? __logf(l) + (m - Elem<T>::get(r[in ? t : 0])) : NAN;
            loss[row] = x;
            if (stats) stats[row] = float2_t{m, in ? 1.f / l : NAN};
            sum += x;
            ++labels;
        }
    }
    if (sums) {
        __shared__ double ss[ROWS];
        __shared__ int ns[ROWS];
        if (tid == 0) { ss[threadIdx.x / LANES] = sum; ns[threadIdx.x / LANES] = labels; }
        __syncthreads();
        if (threadIdx.x == 0 && part * ROWS < N) {
            for (int i = 1; i < ROWS; ++i) { sum += ss[i]; labels += ns[i]; }
            sums[part] = sum;
            counts[part] = labels;
        }
    }
}

// The rows' loss, or its mean over the labels (NaN where there is none), from
// the workgroups' sums, and the factor 1, or 1 / number of labels.
__global__ void __launch_bounds__(1024)
xent_reduce_kernel(const double* __restrict__ sums, const int* __restrict__ counts, int parts,
                   int mean, float* __restrict__ result, float* __restrict__ factor) {
    double s = 0.0;
    int n = 0;
    for (int i0 = threadIdx.x; i0 < parts; i0 += 8 * 1024) {
        // eight on their way at a time, with no branch between them
        double x[8];
        int c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = min(i0 + u * 1024, parts - 1);
            x[u] = sums[i];
            c[u] = counts[i];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * 1024 < parts) {
                s += x[u];
                n += c[u];
            }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        s += __shfl_xor(s, off, WAVE);
        n += __shfl_xor(n, off, WAVE);
    }
    __shared__ double ss[16];
    __shared__ int ns[16];
    if ((threadIdx.x & 63) == 0) { ss[threadIdx.x >> 6] = s; ns[threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) { s += ss[w]; n += ns[w]; }
        *result = (float)(mean ? s / (double)n : s);
        *factor = mean ? (float)(1.0 / (double)n) : 1.f;
    }
}

// `gout`: one value, or one a row (gstride 1).  `factor`: the 1/n of a mean.
// Vectors begin at dx's 16-byte boundaries, and are read wherever that is in x: rows
// of another distance need no copy (128255 columns of 128256, 4096 rows of bf16: loss
// and gradient 0.63 ms; 0.58 for all columns, 0.96 with a copy).
template <typename T, int WAVES>
__global__ void __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64)
xent_bwd_kernel(const T* __restrict__ x, long stride, const long* __restrict__ targets,
                long ignore, int N, int V, const float2_t* __restrict__ stats,
                const float* __restrict__ gout, long gstride,
                const float* __restrict__ factor, T* __restrict__ dx, long dstride) {
    constexpr int VEC = Elem<T>::VEC, LANES = WAVES * 64;
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    constexpr int U = 4;
    const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / LANES;
    if (row >= N) return;
    const int tid = threadIdx.x % LANES;
    const long t = targets[row];
    const T* r = x + row * stride;
    T* d = dx + row * dstride;
    const int head = head_of(d, V);
    const int vecs = (V - head) / VEC;
    const int tail = head + vecs * VEC;
    Vec<T>* out = reinterpret_cast<Vec<T>*>(d + head);
    if (t == ignore) {
        for (int i = tid; i < vecs; i += LANES) out[i] = Vec<T>{};
        if (tid < head) d[tid] = T{};
        if (tail + tid < V) d[tail + tid] = T{};
        return;
    }
    const float2_t st = stats[row];
    const float g = gout[row * gstride] * (factor ? *factor : 1.f);
    const float m = st[0] == -INFINITY ? 0.f : st[0], inv = st[1];
    auto one = [&](int j, float v) {
        return Elem<T>::put((exp_neg<T>(v - m) * inv - (j == t ? 1.f : 0.f)) * g);
    };
    const Loose<T>* body = reinterpret_cast<const Loose<T>*>(r + head);
    auto step = [&](int i0, auto whole) {
        Vec<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = body[whole ? i0 + u * LANES : min(i0 + u * LANES, vecs - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * LANES;
            if (whole || i < vecs) {
                Vec<T> w;
                const int j0 = head + i * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] = one(j0 + j, Elem<T>::get(v[u][j]));
                out[i] = w;
            }
        }
    };
    int i0 = 0;
    for (; i0 + U * LANES <= vecs; i0 += U * LANES) step(i0 + tid, std::true_type{});
    if (i0 < vecs) step(i0 + tid, std::false_type{});
    if (tid < head) d[tid] = one(tid, Elem<T>::get(r[tid]));
    if (tail + tid < V) d[tail + tid] = one(tail + tid, Elem<T>::get(r[tail + tid]));
}

// ---------------------------------------------------------------- launchers
// Each returns the launch's hipError_t.  kind: 0 fp32, 1 bf16, 2 fp16.

namespace {

template <int WAVES> constexpr int rows_of = WAVES < 4 ? 4 / WAVES : 1;

// A launch's threads along x are counted in 32 bits: more workgroups go along y.
template <int WAVES>
dim3 grid_of(int N) {
    const int blocks = (N - 1) / rows_of<WAVES> + 1, most = 1 << 21;
    return blocks <= most ? dim3(blocks) : dim3(most, (blocks - 1) / most + 1);
}

template <typename T, int WAVES>
void fwd(const void* x, long stride, const void* targets, long ignore, int N, int V,
         void* loss, void* stats, void* sums, void* counts, hipStream_t st) {
    constexpr int ROWS = rows_of<WAVES>;
    hipLaunchKernelGGL((xent_fwd_kernel<T, WAVES>), grid_of<WAVES>(N),
                       dim3(ROWS * WAVES * 64), 0, st, (const T*)x, stride,
                       (const long*)targets, ignore, N, V, (float*)loss, (float2_t*)stats,
                       (double*)sums, (int*)counts);
}

template <typename T, int WAVES>
void bwd(const void* x, long stride, const void* targets, long ignore, int N, int V,
         const void* stats, const void* gout, long gstride, const void* factor, void* dx,
         long dstride, hipStream_t st) {
    constexpr int ROWS = rows_of<WAVES>;
    hipLaunchKernelGGL((xent_bwd_kernel<T, WAVES>), grid_of<WAVES>(N),
                       dim3(ROWS * WAVES * 64), 0, st, (const T*)x, stride,
                       (const long*)targets, ignore, N, V, (const float2_t*)stats,
                       (const float*)gout, gstride, (const float*)factor, (T*)dx, dstride);
}

}  // namespace

// How many sums and counts the forward kernel leaves.
extern "C" int xent_parts(int N, int V) {
    const int rows = V <= XENT_SHORT ? rows_of<1> : rows_of<16>;
    return (N - 1) / rows + 1;
}

extern "C" int launch_xent_fwd(int kind, const void* x, long stride, const void* targets,
                               long ignore, int N, int V, void* loss, void* stats, void* sums,
                               void* counts, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
#define FWD(T)                                                                             \
    if (V <= XENT_SHORT)                                                                   \
        fwd<T, 1>(x, stride, targets, ignore, N, V, loss, stats, sums, counts, st);        \
    else                                                                                   \
        fwd<T, 16>(x, stride, targets, ignore, N, V, loss, stats, sums, counts, st)
    if (kind == 0) { FWD(float); }
    else if (kind == 1) { FWD(__bf16); }
    else { FWD(_Float16); }
#undef FWD
    return (int)hipGetLastError();
}

extern "C" int launch_xent_reduce(const void* sums, const void* counts, int parts, int mean,
                                  void* result, void* factor, void* stream) {
    hipLaunchKernelGGL(xent_reduce_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream,
                       (const double*)sums, (const int*)counts, parts, mean, (float*)result,
                       (float*)factor);
    return (int)hipGetLastError();
}

extern "C" int launch_xent_bwd(int kind, const void* x, long stride, const void* targets,
                               long ignore, int N, int V, const void* stats,
                               const void* gout, long gstride, const void* factor, void* dx,
                               long dstride, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
#define BWD(T)                                                                          \
    if (V <= XENT_SHORT)                                                                      \
        bwd<T, 1>(x, stride, targets, ignore, N, V, stats, gout, gstride, factor, dx,   \
                  dstride, st);                                                         \
    else                                                                                \
        bwd<T, 16>(x, stride, targets, ignore, N, V, stats, gout, gstride, factor, dx,  \
                   dstride, st)
    if (kind == 0) { BWD(float); }
    else if (kind == 1) { BWD(__bf16); }
    else { BWD(_Float16); }
#undef BWD
    return (int)hipGetLastError();
}
