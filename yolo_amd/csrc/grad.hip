// The norm of the gradients of many tensors, clipping, and the momentum step on clipped gradients, for gfx950.
//
// What detectron2's SOLVER.CLIP_GRADIENTS wraps around the optimizer (torch.nn.utils.clip_grad_norm_ / clip_grad_value_):
//
//   norm  p = 1: sum |g|,  p = 2: sqrt(sum g * g),  p = inf: max |g|  -- over all tensors, or of each tensor
//   k     = min(1, max_norm / (norm + 1e-6)), one factor or one for each tensor;  g = k * g
//   step  d = k * g (or g clamped to [-v, v]) + wd * w;   m = mu * m + d;   w = w - lr * m
//
// Memory-bound.  A table on the device says which run of which tensor a workgroup owns, so any number of tensors takes one
// launch; a run's sum is fp64 from the first element on (62 million squares leave fp32's range and precision, and the
// conversion and fp64 additions stay hidden behind the loads) and sums are joined in the table's order: no atomics, the same
// result every time.
#include "common.h"

namespace yolo {

constexpr int GRAD_THREADS = 256;

// Loads and stores that go past the caches: 62 million elements in place, or with weights and momentum, are more than the 256 MB
// cache holds, and the gradients that the norm's pass has left in it are worth more than what is written (clipping 248 MB:
// 146 -> 122 us, the step on them 284 -> 222 us; sets of a few MB: the same).
template <typename T>
__device__ __forceinline__ T grad_load(const void* p) { return __builtin_nontemporal_load((const T*)p); }
template <typename T>
__device__ __forceinline__ void grad_store(void* p, const T& v) { __builtin_nontemporal_store(v, (T*)p); }

// p as the kernels know it
enum { GRAD_L1 = 0, GRAD_L2 = 1, GRAD_MAX = 2 };

template <int P>
__device__ __forceinline__ double grad_join(double a, double b) {
    if constexpr (P == GRAD_MAX) return (b > a || b != b) ? b : a;  // a NaN stays
    return a + b;
}
template <int P>
__device__ __forceinline__ double grad_add(double acc, float g) {
    if constexpr (P == GRAD_MAX) return grad_join<P>(acc, (double)fabsf(g));
    if constexpr (P == GRAD_L1) return acc + (double)fabsf(g);
    return acc + (double)g * (double)g;
}

// The join of a workgroup's values, valid in thread 0.
template <int P, int WAVES>
__device__ __forceinline__ double grad_block_join(double v) {
    __shared__ double part[WAVES];
    for (int o = 32; o; o >>= 1) v = grad_join<P>(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < WAVES; ++i) v = grad_join<P>(v, part[i]);
    return v;
}

// f(first element index) for single elements up to a 16-byte boundary and behind the last whole vector, fv for vectors.
template <typename E, typename F, typename FV>
__device__ __forceinline__ void grad_walk(const yolo_grad_block& b, F f, FV fv) {
    constexpr int V = 16 / (int)sizeof(E);
    int head = (int)((16 - ((uintptr_t)b.ptr & 15)) & 15) / (int)sizeof(E);
    if (head > b.count) head = b.count;
    const int vecs = (b.count - head) / V, tail = head + vecs * V;
    if ((int)threadIdx.x < head) f((int)threadIdx.x);
#pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += GRAD_THREADS) fv(head + i * V);
    if (tail + (int)threadIdx.x < b.count) f(tail + (int)threadIdx.x);
}

// partial[run] = the run's sum (or largest value).  Bound by the read: 62 M f32 elements, 248 MB in 45 us, 5.5 TB/s, fp64 additions
// in four chains beside four vectors on their way.  Runs of 16384 elements keep a workgroup's ramp small beside its run; small sets
// get shorter ones so that the CUs are busy (six tensors of 3.1 M elements: 4.0 us).
template <int P>
__global__ void __launch_bounds__(GRAD_THREADS) grad_norm_kernel(const yolo_grad_block* blocks, double* partial) {
    const yolo_grad_block b = blocks[blockIdx.x];
    double acc = 0.0, more[4] = {0.0, 0.0, 0.0, 0.0};  // four chains of additions
    if (b.dtype == YOLO_BF16) {
        const unsigned short* g = (const unsigned short*)b.ptr;
        grad_walk<unsigned short>(
            b, [&](int i) { acc = grad_add<P>(acc, bf16_bits_to_f32(g[i])); },
            [&](int i) {
                const u32x4 v = *(const u32x4*)(g + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    more[e] = grad_add<P>(more[e], __uint_as_float(v[e] << 16));
                    more[e] = grad_add<P>(more[e], __uint_as_float(v[e] & 0xffff0000u));
                }
            });
    } else {
        const float* g = (const float*)b.ptr;
        grad_walk<float>(
            b, [&](int i) { acc = grad_add<P>(acc, g[i]); },
            [&](int i) {
                const f32x4 v = *(const f32x4*)(g + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) more[e] = grad_add<P>(more[e], v[e]);
            });
    }
    for (int e = 0; e < 4; ++e) acc = grad_join<P>(acc, more[e]);
    acc = grad_block_join<P, GRAD_THREADS / 64>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Norm and factor of a sum (or largest value).
template <int P>
__device__ __forceinline__ float grad_factor(double acc, float max_norm, float* norm) {
    *norm = (float)(P == GRAD_L2 ? sqrt(acc) : acc);
    const float k = max_norm / (*norm + 1e-6f);
    return k > 1.f ? 1.f : k;  // a NaN stays
}

// Workgroup t: the runs [first[t], first[t + 1]) -> norm and factor t.  first null: one norm over all n_blocks.  Latency-bound, 2 to
// 4 us.  (The last workgroup to arrive could join instead, but what every workgroup needs for that, a release past its XCD's cache, made
// the norm of 62 M elements 180 us longer.)
template <int P>
__global__ void __launch_bounds__(1024) grad_finish_kernel(const double* partial, const int* first, int n_blocks, float max_norm,
                                                           float* norms, float* coefs) {
    const int t = blockIdx.x, lo = first ? first[t] : 0, hi = first ? first[t + 1] : n_blocks;
    double acc = 0.0;
    for (int i = lo + threadIdx.x; i < hi; i += 1024) acc = grad_join<P>(acc, partial[i]);
    acc = grad_block_join<P, 16>(acc);
    if (threadIdx.x == 0) {
        float norm;
        const float k = grad_factor<P>(acc, max_norm, &norm);
        norms[t] = norm;
        if (coefs) coefs[t] = k;
    }
}

// MODE 0: g = k * g;  MODE 1: g clamped to [-v, v] (a NaN stays)
template <int MODE>
__device__ __forceinline__ float grad_clip(float g, float k) {
    if constexpr (MODE == 0) return g * k;
    return g > k ? k : (g < -k ? -k : g);
}

template <int MODE>
__device__ __forceinline__ void grad_clip_run(const yolo_grad_block& b, float k) {
    if (b.dtype == YOLO_BF16) {
        unsigned short* g = (unsigned short*)b.ptr;
        grad_walk<unsigned short>(
            b, [&](int i) { g[i] = f32_to_bf16_bits(grad_clip<MODE>(bf16_bits_to_f32(g[i]), k)); },
            [&](int i) {
                u32x4 v = grad_load<u32x4>(g + i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = pack_bf16x2(grad_clip<MODE>(__uint_as_float(v[e] << 16), k),
                                       grad_clip<MODE>(__uint_as_float(v[e] & 0xffff0000u), k));
                grad_store(g + i, v);
            });
    } else {
        float* g = (float*)b.ptr;
        grad_walk<float>(
            b, [&](int i) { g[i] = grad_clip<MODE>(g[i], k); },
            [&](int i) {
                f32x4 v = grad_load<f32x4>(g + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = grad_clip<MODE>(v[e], k);
                grad_store(g + i, v);
            });
    }
}

// In place; 62 M f32 elements: 496 MB in 72 us, 6.9 TB/s, of which the norm's pass has left part in the cache.  bf16 products are
// rounded once, to the gradient's own type.
template <int MODE>
__global__ void __launch_bounds__(GRAD_THREADS) grad_clip_kernel(const yolo_grad_block* blocks, const float* coefs, int per_tensor,
                                                                 float value) {
    const yolo_grad_block b = blocks[blockIdx.x];
    grad_clip_run<MODE>(b, MODE == 0 ? coefs[per_tensor ? b.tensor : 0] : value);
}

// grad_finish_kernel and the product in one launch, for at most GRAD_JOIN runs: every workgroup joins the sums for itself, in the
// order of grad_finish_kernel (a thread stands for four of its threads), so that both give the same bits.  Six tensors of 3.1 M
// elements: 14.0 -> 10.0 us a call.  With the 3900 runs of 62 M elements each workgroup would read 31 KB of sums for its 64 KB run.
constexpr int GRAD_JOIN = 1024;
template <int P>
__global__ void __launch_bounds__(GRAD_THREADS) grad_join_clip_kernel(const yolo_grad_block* blocks, const double* partial,
                                                                      const int* first, int n_tensors, int n_blocks, float max_norm,
                                                                      float* norms, float* coefs) {
    __shared__ double part[16];
    const yolo_grad_block b = blocks[blockIdx.x];
    const int t = first ? b.tensor : 0, lo = first ? first[t] : 0, hi = first ? first[t + 1] : n_blocks;
    double v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = lo + (int)threadIdx.x + j * GRAD_THREADS;
        v[j] = i < hi ? grad_join<P>(0.0, partial[i]) : 0.0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        for (int o = 32; o; o >>= 1) v[j] = grad_join<P>(v[j], __shfl_xor(v[j], o));
        if ((threadIdx.x & 63) == 0) part[(threadIdx.x >> 6) + 4 * j] = v[j];
    }
    __syncthreads();
    double acc = part[0];
    for (int i = 1; i < 16; ++i) acc = grad_join<P>(acc, part[i]);
    float norm;
    const float k = grad_factor<P>(acc, max_norm, &norm);
    if ((int)blockIdx.x == lo && threadIdx.x == 0) {
        norms[t] = norm;
        coefs[t] = k;
    }
    if (first && blockIdx.x == 0)  // tensors without elements have no run that would write theirs
        for (int i = threadIdx.x; i < n_tensors; i += GRAD_THREADS)
            if (first[i] == first[i + 1]) coefs[i] = grad_factor<P>(0.0, max_norm, &norms[i]);
    grad_clip_run<0>(b, k);
}

struct SgdClipParams {
    float* param;
    const float* grad;
    float* mom;
    const int* blocks;   // [n][4]: first element, count, group, tensor
    const float* coefs;  // null: clamp to [-value, value]
    int per_tensor;
    float lr[2], wd[2];
    float momentum, value;
};

// One launch over the arenas; 62 M weights: 1.24 GB in 175 us, 7.1 TB/s.  The clipped gradient exists in a register only: writing it
// back first and reading it again would be 496 MB more.  Runs of 4096 elements: a weight moves 20 bytes, and their ends are aligned.
__global__ void __launch_bounds__(GRAD_THREADS) sgd_step_clipped_kernel(const SgdClipParams p) {
    const int first = p.blocks[4 * blockIdx.x], count = p.blocks[4 * blockIdx.x + 1], g = p.blocks[4 * blockIdx.x + 2];
    const bool scale = p.coefs != nullptr;
    const float k = scale ? p.coefs[p.per_tensor ? p.blocks[4 * blockIdx.x + 3] : 0] : p.value;
    const float lr = p.lr[g], wd = p.wd[g], mu = p.momentum;
    float* w = p.param + first;
    float* m = p.mom + first;
    const float* d = p.grad + first;
    auto one = [&](float& wv, float& mv, float dv) {
        dv = scale ? grad_clip<0>(dv, k) : grad_clip<1>(dv, k);
        if (wd != 0.f) dv = dv + wd * wv;
        mv = mv * mu + dv;
        wv = wv - lr * mv;
    };
    // the three arenas have one layout: their runs begin at the same distance from a 16-byte boundary
    int head = (4 - (first & 3)) & 3;
    if (head > count) head = count;
    const int vecs = (count - head) / 4, tail = head + vecs * 4;
    auto single = [&](int i) {
        float wv = w[i], mv = m[i];
        one(wv, mv, d[i]);
        m[i] = mv;
        w[i] = wv;
    };
    if ((int)threadIdx.x < head) single((int)threadIdx.x);
#pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += GRAD_THREADS) {
        const int at = head + i * 4;
        f32x4 wv = grad_load<f32x4>(w + at), mv = grad_load<f32x4>(m + at);
        const f32x4 dv = grad_load<f32x4>(d + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a = wv[e], b = mv[e];
            one(a, b, dv[e]);
            wv[e] = a;
            mv[e] = b;
        }
        grad_store(m + at, mv);
        grad_store(w + at, wv);
    }
    if (tail + (int)threadIdx.x < count) single(tail + (int)threadIdx.x);
}

}  // namespace yolo

using namespace yolo;

extern "C" size_t yolo_grad_norm_workspace_bytes(int n_blocks) { return n_blocks > 0 ? (size_t)n_blocks * sizeof(double) : 16; }

static int grad_norm_launch(const char* op, bool clip, const yolo_grad_block* blocks, int n_blocks, const int* tensor_first, int n_tensors,
                            float norm_type, float max_norm, float* norms, float* coefs, void* workspace, size_t ws_bytes, hipStream_t st) {
    YOLO_REQUIRE(norms && workspace && (blocks || n_blocks == 0) && (coefs || !clip), "%s: null argument", op);
    YOLO_REQUIRE(n_blocks >= 0, "%s: %d blocks", op, n_blocks);
    YOLO_REQUIRE(!tensor_first || n_tensors > 0, "%s: a norm for each of %d tensors", op, n_tensors);
    YOLO_REQUIRE((uintptr_t)workspace % 16 == 0, "%s: workspace is not 16-byte aligned", op);
    YOLO_REQUIRE(norm_type == 1.f || norm_type == 2.f || (__builtin_isinf(norm_type) && norm_type > 0.f),
                 "%s: norm type %g (1, 2 and inf are built)", op, (double)norm_type);
    YOLO_REQUIRE(!coefs || max_norm >= 0.f, "%s: max_norm %g", op, (double)max_norm);
    if (ws_bytes < yolo_grad_norm_workspace_bytes(n_blocks))
        return fail(YOLO_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, ws_bytes, yolo_grad_norm_workspace_bytes(n_blocks));
    double* partial = (double*)workspace;
    const unsigned outs = tensor_first ? (unsigned)n_tensors : 1u;
    auto apart = [](const void* a, size_t an, const void* b, size_t bn) {
        return !a || !b || (uintptr_t)a + an <= (uintptr_t)b || (uintptr_t)b + bn <= (uintptr_t)a;
    };
    YOLO_REQUIRE(apart(norms, outs * 4ull, coefs, outs * 4ull) && apart(norms, outs * 4ull, partial, n_blocks * 8ull) &&
                     apart(coefs, outs * 4ull, partial, n_blocks * 8ull),
                 "%s: norms, factors and workspace share memory", op);
    const dim3 runs((unsigned)n_blocks);
#define GRAD_NORM(P)                                                                                                             \
    do {                                                                                                                         \
        if (n_blocks) hipLaunchKernelGGL((grad_norm_kernel<P>), runs, dim3(GRAD_THREADS), 0, st, blocks, partial);               \
        if (clip && n_blocks && n_blocks <= GRAD_JOIN) {                                                                         \
            hipLaunchKernelGGL((grad_join_clip_kernel<P>), runs, dim3(GRAD_THREADS), 0, st, blocks, partial, tensor_first,       \
                               n_tensors, n_blocks, max_norm, norms, coefs);                                                     \
            break;                                                                                                               \
        }                                                                                                                        \
        hipLaunchKernelGGL((grad_finish_kernel<P>), dim3(outs), dim3(1024), 0, st, partial, tensor_first, n_blocks, max_norm,    \
                           norms, coefs);                                                                                        \
        if (clip && n_blocks)                                                                                                    \
            hipLaunchKernelGGL((grad_clip_kernel<0>), runs, dim3(GRAD_THREADS), 0, st, blocks, coefs, tensor_first != nullptr,   \
                               0.f);                                                                                             \
    } while (0)
    if (norm_type == 2.f)
        GRAD_NORM(GRAD_L2);
    else if (norm_type == 1.f)
        GRAD_NORM(GRAD_L1);
    else
        GRAD_NORM(GRAD_MAX);
#undef GRAD_NORM
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}

extern "C" int yolo_grad_norm(const yolo_grad_block* blocks, int n_blocks, const int* tensor_first, int n_tensors,
                              float norm_type, float max_norm, float* norms, float* coefs, void* workspace, size_t ws_bytes,
                              void* stream) {
    return grad_norm_launch("grad_norm", false, blocks, n_blocks, tensor_first, n_tensors, norm_type, max_norm, norms, coefs, workspace,
                            ws_bytes, (hipStream_t)stream);
}

extern "C" int yolo_grad_clip(const yolo_grad_block* blocks, int n_blocks, const int* tensor_first, int n_tensors,
                              float norm_type, float max_norm, float* norms, float* coefs, void* workspace, size_t ws_bytes,
                              void* stream) {
    return grad_norm_launch("grad_clip", true, blocks, n_blocks, tensor_first, n_tensors, norm_type, max_norm, norms, coefs, workspace,
                            ws_bytes, (hipStream_t)stream);
}

extern "C" int yolo_grad_clamp(const yolo_grad_block* blocks, int n_blocks, float value, void* stream) {
    YOLO_REQUIRE(n_blocks >= 0 && (blocks || n_blocks == 0), "grad_clamp: bad argument");
    YOLO_REQUIRE(value >= 0.f, "grad_clamp: value %g", (double)value);
    if (n_blocks == 0) return YOLO_OK;
    hipLaunchKernelGGL((grad_clip_kernel<1>), dim3((unsigned)n_blocks), dim3(GRAD_THREADS), 0, (hipStream_t)stream, blocks, nullptr, 0,
                       value);
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}

extern "C" int yolo_sgd_step_clipped(float* param, const float* grad, float* momentum_buf, const int* block_table, int n_blocks,
                                     float lr0, float weight_decay0, float lr1, float weight_decay1, float momentum,
                                     const float* coefs, int per_tensor, float clip_value, void* stream) {
    YOLO_REQUIRE(param && grad && momentum_buf && block_table && n_blocks > 0, "sgd_step_clipped: bad argument");
    YOLO_REQUIRE(coefs || clip_value >= 0.f, "sgd_step_clipped: clip value %g", (double)clip_value);
    YOLO_REQUIRE((uintptr_t)param % 16 == 0 && (uintptr_t)grad % 16 == 0 && (uintptr_t)momentum_buf % 16 == 0,
                 "sgd_step_clipped: the arenas have to begin at 16-byte boundaries");
    SgdClipParams p{};
    p.param = param;
    p.grad = grad;
    p.mom = momentum_buf;
    p.blocks = block_table;
    p.coefs = coefs;
    p.per_tensor = per_tensor;
    p.lr[0] = lr0;
    p.lr[1] = lr1;
    p.wd[0] = weight_decay0;
    p.wd[1] = weight_decay1;
    p.momentum = momentum;
    p.value = clip_value;
    hipLaunchKernelGGL(sgd_step_clipped_kernel, dim3(n_blocks), dim3(GRAD_THREADS), 0, (hipStream_t)stream, p);
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}
