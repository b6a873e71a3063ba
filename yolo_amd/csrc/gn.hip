// Group normalisation + activation (+ residual) of pixel-major activations, forward and backward, for gfx950.
//
// What detectron2's get_norm("GN") puts behind every Conv2d (yolo/modeling/backbone/darknet.py:45-53,74-106, fpn.py:23-30,
// 44-61,78-90 take the norm's name from the config) and the F.leaky_relu after it, with their autograd backward.
//
//   forward   mean, var over the H*W*Cg values of an (image, group);  r = 1 / sqrt(var + eps)
//             t = (x - mean) * r * gamma + beta;   y = act(t) [+ residual];   mean and r are kept
//   backward  d = dy * act'(t),  xh = (x - mean) * r,  M = H*W*Cg
//             dbeta = sum over images and pixels of d,  dgamma = the same of d * xh
//             dx = r * (gamma * d - A - xh * B),  A = sum over the group of gamma * d / M,  B = the same of d * xh
//
// Memory-bound: a pass reads or writes 16 bytes per lane, sums are fp32 within a thread (about a pivot where squares would
// cancel) and fp64 from there on.
#include "common.h"

namespace yolo {

struct GnTensor {
    char* p;        // logical pixel (0, 0), first channel of the view, image 0
    long long img;  // bytes between images
    int row, pix;   // bytes between rows, between pixels
};

struct GnParams {
    GnTensor x, r, dy, y;  // r: residual (p null: none); y: forward output, backward dx
    int N, H, W, HW, C, Cg, groups;
    int VS, PL;            // 16-byte vectors of a slab, pixel lanes of a workgroup
    int chunk, chunks;     // pixels of a workgroup, workgroups of an image's slab
    const float* gamma;
    const float* beta;
    float* stats;          // [2][N][groups]: mean, r
    float* dgamma;
    float* dbeta;
    void* partial;         // forward: double [N][chunks][2][C]; backward: float [N][chunks][2][C]
    float* sums;           // backward: [N][2][C], one image's sums of d and of d * xh
    float* terms;          // backward: [2][N][groups], A and B
    float eps, slope;
    double inv_count;      // 1 / M
};

constexpr int GN_THREADS = 256;
constexpr int GN_MAX_CHUNKS = 64;

template <typename E> struct GnVec;
template <> struct GnVec<unsigned short> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const u32x4& r, float* v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(r[e] << 16);
            v[2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float* v) {
        return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    }
};
template <> struct GnVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const u32x4& r, float* v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(r[e]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* v) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
};

// A position in an image, moved on by a fixed number of pixels without divisions.
struct GnCursor {
    int h, w, sh, sw, W;
    __device__ __forceinline__ GnCursor(int pixel, int step, int W_) : W(W_) {
        h = pixel / W;
        w = pixel - h * W;
        sh = step / W;
        sw = step - sh * W;
    }
    __device__ __forceinline__ void next() {
        w += sw;
        h += sh;
        if (w >= W) {
            w -= W;
            ++h;
        }
    }
    __device__ __forceinline__ int at(const GnTensor& t) const { return h * t.row + w * t.pix; }
};

constexpr int GN_LEAKY = YOLO_ACT_LEAKY, GN_SILU = YOLO_ACT_SILU;

// exp through v_exp_f32 and a 1-ulp reciprocal: both are within a few 2^-24 of the value, far inside what the sums around
// them keep.  t = -inf and +inf give 0 and 1.
__device__ __forceinline__ float gn_sigmoid(float t) { return __builtin_amdgcn_rcpf(1.f + __expf(-t)); }

template <int ACT>
__device__ __forceinline__ float gn_act(float t, float slope) {
    if constexpr (ACT == GN_SILU) return t * gn_sigmoid(t);
    return t > 0.f ? t : t * slope;
}

// d = dy * act'(t) with t = xh * gamma + beta.  The leaky derivative jumps at t = 0 (slope at t == 0, torch's convention), so
// the side is decided exactly: fp32 rounds t by less than 2^-22 (|beta| + |t|) -- three roundings of xh * gamma, which is
// about -beta there, and one of the sum -- and a t nearer to zero than 2^-20 |beta| is computed again in fp64.  One value in
// about a million takes that branch.
template <int ACT>
__device__ __forceinline__ float gn_act_grad(float dy, float x, float xh, float mean, float r, float gamma, float beta, float slope) {
    const float t = xh * gamma + beta;
    if constexpr (ACT == GN_SILU) {
        const float s = gn_sigmoid(t);
        return dy * (s * (1.f + t * (1.f - s)));
    } else {
        bool up = t > 0.f;
        if (__builtin_expect(fabsf(t) <= fabsf(beta) * 0x1p-20f, 0))
            up = ((double)x - (double)mean) * (double)r * (double)gamma + (double)beta > 0.0;
        return up ? dy : dy * slope;
    }
}

// Which vector and pixel lane a thread has: the vectors of a pixel are next to each other in a wave.
struct GnLane {
    int pl, c;  // pixel lane; first channel of the vector
    bool on;
};
template <typename E>
__device__ __forceinline__ GnLane gn_lane(const GnParams& p) {
    GnLane l;
    const int v = threadIdx.x % p.VS;
    l.pl = threadIdx.x / p.VS;
    l.c = (blockIdx.y * p.VS + v) * GnVec<E>::N;
    l.on = l.pl < p.PL && l.c < p.C;
    return l;
}

// ------------------------------------------------------------------------------------------------ forward, sums
// partial[n][chunk][0 / 1][c] = sum of x, of x * x over the chunk's pixels.  A thread sums differences from the first value
// it sees (fp32; the values of a few dozen pixels differ from it by about their spread), and goes over to fp64 after that.
template <typename E>
__global__ void __launch_bounds__(GN_THREADS) gn_sums_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ double red[GN_THREADS * V];
    const GnLane l = gn_lane<E>(p);
    const int n = blockIdx.z, first = blockIdx.x * p.chunk, last = min(first + p.chunk, p.HW);
    const char* base = p.x.p + n * p.x.img + l.c * (int)sizeof(E);
    float k[V], s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
    int count = 0;
    if (l.on && first + l.pl < last) {
        GnCursor c(first + l.pl, p.PL, p.W);
        count = (last - first - l.pl + p.PL - 1) / p.PL;
        GnVec<E>::unpack(*(const u32x4*)(base + c.at(p.x)), k);
        c.next();
#pragma unroll 4
        for (int i = 1; i < count; ++i) {
            float v[V];
            GnVec<E>::unpack(*(const u32x4*)(base + c.at(p.x)), v);
            c.next();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = v[e] - k[e];
                s[e] += d;
                q[e] += d * d;
            }
        }
    }
    const int S = p.VS * V;
    double* out = (double*)p.partial + (((long long)n * p.chunks + blockIdx.x) * 2) * p.C + blockIdx.y * S;
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double K = k[e], sd = s[e];
            red[threadIdx.x * V + e] = which == 0 ? count * K + sd : (double)q[e] + K * (2.0 * sd + count * K);
        }
        __syncthreads();
        for (int j = threadIdx.x; j < S && blockIdx.y * S + j < p.C; j += GN_THREADS) {
            double a = 0.0;
            for (int i = 0; i < p.PL; ++i) a += red[i * S + j];
            out[(long long)which * p.C + j] = a;
        }
        __syncthreads();
    }
}

// One workgroup per (group, image): chunk sums -> mean and r.
__global__ void __launch_bounds__(64) gn_stats_kernel(const GnParams p) {
    const int g = blockIdx.x, n = blockIdx.y, total = p.chunks * p.Cg;
    const double* part = (const double*)p.partial + (long long)n * p.chunks * 2 * p.C + g * p.Cg;
    double s = 0.0, q = 0.0;
    for (int i = threadIdx.x; i < total; i += 64) {
        const int ch = i / p.Cg, c = i - ch * p.Cg;
        s += part[(long long)ch * 2 * p.C + c];
        q += part[((long long)ch * 2 + 1) * p.C + c];
    }
    for (int o = 32; o; o >>= 1) {
        s += __shfl_xor(s, o);
        q += __shfl_xor(q, o);
    }
    if (threadIdx.x == 0) {
        const double mean = s * p.inv_count;
        double var = q * p.inv_count - mean * mean;
        var = var < 0.0 ? 0.0 : var;
        p.stats[n * p.groups + g] = (float)mean;
        p.stats[(p.N + n) * p.groups + g] = (float)(1.0 / sqrt(var + (double)p.eps));
    }
}

// ------------------------------------------------------------------------------------------------ forward, output
template <typename E, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_apply_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    const GnLane l = gn_lane<E>(p);
    // the pass before this one walked forwards: its last chunks are the ones still in the caches
    const int n = p.N - 1 - blockIdx.z, chunk = p.chunks - 1 - blockIdx.x;
    const int first = chunk * p.chunk, last = min(first + p.chunk, p.HW);
    if (!l.on || first + l.pl >= last) return;
    float mean[V], sc[V], beta[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (l.c + e) / p.Cg;
        mean[e] = p.stats[n * p.groups + g];
        sc[e] = p.gamma[l.c + e] * p.stats[(p.N + n) * p.groups + g];
        beta[e] = p.beta[l.c + e];
    }
    const int cb = l.c * (int)sizeof(E);
    const char* x = p.x.p + n * p.x.img + cb;
    const char* r = p.r.p ? p.r.p + n * p.r.img + cb : nullptr;
    char* y = p.y.p + n * p.y.img + cb;
    const int count = (last - first - l.pl + p.PL - 1) / p.PL;
    GnCursor c(first + l.pl, p.PL, p.W);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
        float v[V];
        GnVec<E>::unpack(*(const u32x4*)(x + c.at(p.x)), v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = gn_act<ACT>((v[e] - mean[e]) * sc[e] + beta[e], p.slope);
        if (r) {
            float a[V];
            GnVec<E>::unpack(*(const u32x4*)(r + c.at(p.r)), a);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += a[e];
        }
        *(u32x4*)(y + c.at(p.y)) = GnVec<E>::pack(v);
        c.next();
    }
}

// ------------------------------------------------------------------------------------------------ backward, sums
// partial[n][chunk][0 / 1][c] = sum of d, of d * xh over the chunk's pixels
template <typename E, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_bwd_sums_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ float red[2][GN_THREADS * V];
    const GnLane l = gn_lane<E>(p);
    const int n = blockIdx.z, first = blockIdx.x * p.chunk, last = min(first + p.chunk, p.HW);
    float sd[V], sx[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sd[e] = sx[e] = 0.f;
    if (l.on && first + l.pl < last) {
        float mean[V], is[V], gamma[V], beta[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = (l.c + e) / p.Cg;
            mean[e] = p.stats[n * p.groups + g];
            is[e] = p.stats[(p.N + n) * p.groups + g];
            gamma[e] = p.gamma[l.c + e];
            beta[e] = p.beta[l.c + e];
        }
        const int cb = l.c * (int)sizeof(E);
        const char* x = p.x.p + n * p.x.img + cb;
        const char* dy = p.dy.p + n * p.dy.img + cb;
        const int count = (last - first - l.pl + p.PL - 1) / p.PL;
        GnCursor c(first + l.pl, p.PL, p.W);
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
            float v[V], d[V];
            GnVec<E>::unpack(*(const u32x4*)(x + c.at(p.x)), v);
            GnVec<E>::unpack(*(const u32x4*)(dy + c.at(p.dy)), d);
            c.next();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (v[e] - mean[e]) * is[e];
                const float a = gn_act_grad<ACT>(d[e], v[e], xh, mean[e], is[e], gamma[e], beta[e], p.slope);
                sd[e] += a;
                sx[e] += a * xh;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        red[0][threadIdx.x * V + e] = sd[e];
        red[1][threadIdx.x * V + e] = sx[e];
    }
    __syncthreads();
    const int S = p.VS * V;
    float* out = (float*)p.partial + (((long long)n * p.chunks + blockIdx.x) * 2) * p.C + blockIdx.y * S;
    for (int j = threadIdx.x; j < S && blockIdx.y * S + j < p.C; j += GN_THREADS) {
        float a = 0.f, b = 0.f;
        for (int i = 0; i < p.PL; ++i) {
            a += red[0][i * S + j];
            b += red[1][i * S + j];
        }
        out[j] = a;
        out[p.C + j] = b;
    }
}

// One workgroup per (group, image): chunk sums -> the image's sums per channel and the group's two terms.
__global__ void __launch_bounds__(256) gn_bwd_terms_kernel(const GnParams p) {
    __shared__ double ra[4], rb[4];
    const int g = blockIdx.x, n = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float* part = (const float*)p.partial + (long long)n * p.chunks * 2 * p.C;
    double A = 0.0, B = 0.0;
    for (int j = wave; j < p.Cg; j += 4) {
        const int c = g * p.Cg + j;
        double a = 0.0, b = 0.0;
        for (int i = lane; i < p.chunks; i += 64) {
            a += (double)part[(long long)i * 2 * p.C + c];
            b += (double)part[((long long)i * 2 + 1) * p.C + c];
        }
        for (int o = 32; o; o >>= 1) {
            a += __shfl_xor(a, o);
            b += __shfl_xor(b, o);
        }
        const double gamma = p.gamma[c];
        A += gamma * a;
        B += gamma * b;
        if (lane == 0) {
            p.sums[((long long)n * 2) * p.C + c] = (float)a;
            p.sums[((long long)n * 2 + 1) * p.C + c] = (float)b;
        }
    }
    if (lane == 0) {
        ra[wave] = A;
        rb[wave] = B;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        A = ra[0] + ra[1] + ra[2] + ra[3];
        B = rb[0] + rb[1] + rb[2] + rb[3];
        p.terms[n * p.groups + g] = (float)(A * p.inv_count);
        p.terms[(p.N + n) * p.groups + g] = (float)(B * p.inv_count);
    }
}

// dgamma, dbeta: the images' sums, in their order.
__global__ void __launch_bounds__(256) gn_bwd_params_kernel(const GnParams p) {
    const int i = blockIdx.x * 256 + threadIdx.x;  // [0, 2C): d sums, then d * xh sums
    if (i >= 2 * p.C) return;
    double a = 0.0;
    for (int n = 0; n < p.N; ++n) a += (double)p.sums[(long long)n * 2 * p.C + i];
    if (i < p.C)
        p.dbeta[i] = (float)a;
    else
        p.dgamma[i - p.C] = (float)a;
}

// ------------------------------------------------------------------------------------------------ backward, output
template <typename E, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_bwd_apply_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    const GnLane l = gn_lane<E>(p);
    const int n = p.N - 1 - blockIdx.z, chunk = p.chunks - 1 - blockIdx.x;
    const int first = chunk * p.chunk, last = min(first + p.chunk, p.HW);
    if (!l.on || first + l.pl >= last) return;
    float mean[V], is[V], gamma[V], beta[V], A[V], B[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (l.c + e) / p.Cg;
        mean[e] = p.stats[n * p.groups + g];
        is[e] = p.stats[(p.N + n) * p.groups + g];
        A[e] = p.terms[n * p.groups + g];
        B[e] = p.terms[(p.N + n) * p.groups + g];
        gamma[e] = p.gamma[l.c + e];
        beta[e] = p.beta[l.c + e];
    }
    const int cb = l.c * (int)sizeof(E);
    const char* x = p.x.p + n * p.x.img + cb;
    const char* dy = p.dy.p + n * p.dy.img + cb;
    char* y = p.y.p + n * p.y.img + cb;
    const int count = (last - first - l.pl + p.PL - 1) / p.PL;
    GnCursor c(first + l.pl, p.PL, p.W);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
        float v[V], d[V];
        GnVec<E>::unpack(*(const u32x4*)(x + c.at(p.x)), v);
        GnVec<E>::unpack(*(const u32x4*)(dy + c.at(p.dy)), d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float xh = (v[e] - mean[e]) * is[e];
            const float a = gn_act_grad<ACT>(d[e], v[e], xh, mean[e], is[e], gamma[e], beta[e], p.slope);
            // the products are rounded one by one: with a single value in the group the terms cancel exactly
            v[e] = ((gamma[e] * a - A[e]) - xh * B[e]) * is[e];
        }
        *(u32x4*)(y + c.at(p.y)) = GnVec<E>::pack(v);
        c.next();
    }
}

// ------------------------------------------------------------------------------------------------ host
static int gn_check_view(const yolo_view* v, const yolo_view* like, int N, int C, int es, const char* op, const char* what) {
    YOLO_REQUIRE(v && v->ptr, "%s: %s is null", op, what);
    YOLO_REQUIRE(v->H > 0 && v->W > 0 && v->halo >= 0 && v->H == like->H && v->W == like->W, "%s: %s is %d x %d (halo %d), expected %d x %d",
                 op, what, v->H, v->W, v->halo, like->H, like->W);
    YOLO_REQUIRE(v->ch_offset >= 0 && v->ch_offset % 8 == 0 && v->ch_total % 8 == 0 && v->ch_offset + C <= v->ch_total,
                 "%s: %s: needs an 8-aligned slice of %d channels", op, what, C);
    YOLO_REQUIRE((uintptr_t)v->ptr % 16 == 0, "%s: %s is not 16-byte aligned", op, what);
    YOLO_REQUIRE((long long)(v->H + 2 * v->halo) * (v->W + 2 * v->halo) * v->ch_total * es < (1ll << 31),
                 "%s: %s: one image has to be below 2 GiB", op, what);
    return YOLO_OK;
}

static GnTensor gn_tensor(const yolo_view* v, int es) {
    const ViewGeom g = geom_of(*v);
    return GnTensor{(char*)v->ptr + (long long)g.origin * es, g.img_stride * es, g.row_stride * es, g.pix_stride * es};
}

static int gn_check_shape(int N, int C, int groups, int act, float slope, int dtype, const char* op) {
    YOLO_REQUIRE(dtype == YOLO_F32 || dtype == YOLO_BF16, "%s: dtype %d", op, dtype);
    YOLO_REQUIRE(N > 0 && N <= 65535, "%s: batch %d (1 to 65535)", op, N);
    YOLO_REQUIRE(C > 0 && C % 8 == 0 && C <= 65536, "%s: %d channels (a multiple of 8, at most 65536)", op, C);
    YOLO_REQUIRE(groups > 0 && C % groups == 0, "%s: %d groups do not divide %d channels", op, groups, C);
    YOLO_REQUIRE(act == YOLO_ACT_LEAKY || act == YOLO_ACT_SILU, "%s: activation %d", op, act);
    YOLO_REQUIRE(act != YOLO_ACT_LEAKY || (slope >= 0.f && slope <= 1.f), "%s: leaky slope %g outside [0, 1]", op, (double)slope);
    return YOLO_OK;
}

// The split of an image over workgroups: pixel chunks so that about 2048 workgroups (8 per CU) are there, but no more than 64
// chunks and no fewer than 4 pixels to a thread.
static void gn_split(GnParams& p, int es) {
    const int vecs = p.C * es / 16;
    p.VS = vecs < GN_THREADS ? vecs : GN_THREADS;
    p.PL = GN_THREADS / p.VS;
    const int slabs = (vecs + p.VS - 1) / p.VS;
    long long want = 2048 / ((long long)p.N * slabs);
    if (want < 1) want = 1;
    if (want > GN_MAX_CHUNKS) want = GN_MAX_CHUNKS;
    long long chunk = (p.HW + want - 1) / want;
    if (chunk < 4ll * p.PL) chunk = 4ll * p.PL;
    p.chunk = (int)chunk;
    p.chunks = (int)((p.HW + chunk - 1) / chunk);
}

static dim3 gn_grid(const GnParams& p, int es) {
    const int vecs = p.C * es / 16;
    return dim3(p.chunks, (vecs + p.VS - 1) / p.VS, p.N);
}

static void gn_shape(GnParams& p, const yolo_view* x, int N, int C, int groups, int es) {
    p.N = N;
    p.H = x->H;
    p.W = x->W;
    p.HW = x->H * x->W;
    p.C = C;
    p.groups = groups;
    p.Cg = C / groups;
    p.inv_count = 1.0 / ((double)p.HW * p.Cg);
    gn_split(p, es);
}

}  // namespace yolo

using namespace yolo;

#define GN_LAUNCH(KERNEL, grid, st, p)                                                                                  \
    do {                                                                                                                \
        if (dtype == YOLO_BF16 && act == YOLO_ACT_LEAKY)                                                                \
            hipLaunchKernelGGL((KERNEL<unsigned short, GN_LEAKY>), grid, dim3(GN_THREADS), 0, st, p);                   \
        else if (dtype == YOLO_BF16)                                                                                    \
            hipLaunchKernelGGL((KERNEL<unsigned short, GN_SILU>), grid, dim3(GN_THREADS), 0, st, p);                    \
        else if (act == YOLO_ACT_LEAKY)                                                                                 \
            hipLaunchKernelGGL((KERNEL<float, GN_LEAKY>), grid, dim3(GN_THREADS), 0, st, p);                            \
        else                                                                                                            \
            hipLaunchKernelGGL((KERNEL<float, GN_SILU>), grid, dim3(GN_THREADS), 0, st, p);                             \
    } while (0)

extern "C" size_t yolo_gn_workspace_bytes(int N, int H, int W, int C, int groups, int dtype) {
    if (N <= 0 || H <= 0 || W <= 0 || C <= 0 || C % 8 || groups <= 0 || C % groups || (long long)H * W >= (1ll << 31)) return 0;
    GnParams p{};
    yolo_view v{nullptr, H, W, 0, C, 0};
    gn_shape(p, &v, N, C, groups, (int)elem_size(dtype));
    // forward: the double sums; backward: the float sums, then the images' sums and the groups' terms
    const size_t fwd = (size_t)N * p.chunks * 2 * C * sizeof(double);
    const size_t bwd = ((size_t)N * p.chunks * 2 * C + (size_t)N * 2 * C + (size_t)2 * N * groups) * sizeof(float);
    return fwd > bwd ? fwd : bwd;
}

extern "C" int yolo_gn_act_fwd(const yolo_view* x, const float* gamma, const float* beta, const yolo_view* residual,
                               const yolo_view* y, float* stats, int N, int C, int groups, float eps, int act,
                               float leaky_slope, int dtype, void* workspace, size_t ws_bytes, void* stream) {
    YOLO_REQUIRE(x && gamma && beta && stats && workspace, "gn_act_fwd: null argument");
    if (int e = gn_check_shape(N, C, groups, act, leaky_slope, dtype, "gn_act_fwd")) return e;
    YOLO_REQUIRE(eps >= 0.f, "gn_act_fwd: eps %g is negative", (double)eps);
    const int es = (int)elem_size(dtype);
    if (int e = gn_check_view(x, x, N, C, es, "gn_act_fwd", "x")) return e;
    if (int e = gn_check_view(y, x, N, C, es, "gn_act_fwd", "y")) return e;
    if (residual)
        if (int e = gn_check_view(residual, x, N, C, es, "gn_act_fwd", "residual")) return e;
    YOLO_REQUIRE((uintptr_t)workspace % 16 == 0, "gn_act_fwd: workspace is not 16-byte aligned");
    if (ws_bytes < yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype))
        return fail(YOLO_E_WORKSPACE, "gn_act_fwd: workspace of %zu bytes, %zu needed", ws_bytes,
                    yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype));
    GnParams p{};
    gn_shape(p, x, N, C, groups, es);
    p.x = gn_tensor(x, es);
    p.y = gn_tensor(y, es);
    if (residual) p.r = gn_tensor(residual, es);
    p.gamma = gamma;
    p.beta = beta;
    p.stats = stats;
    p.partial = workspace;
    p.eps = eps;
    p.slope = leaky_slope;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid = gn_grid(p, es);
    if (dtype == YOLO_BF16)
        hipLaunchKernelGGL((gn_sums_kernel<unsigned short>), grid, dim3(GN_THREADS), 0, st, p);
    else
        hipLaunchKernelGGL((gn_sums_kernel<float>), grid, dim3(GN_THREADS), 0, st, p);
    hipLaunchKernelGGL(gn_stats_kernel, dim3(groups, N), dim3(64), 0, st, p);
    GN_LAUNCH(gn_apply_kernel, grid, st, p);
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}

extern "C" int yolo_gn_act_bwd(const yolo_view* dy, const yolo_view* x, const float* gamma, const float* beta,
                               const float* stats, const yolo_view* dx, float* dgamma, float* dbeta, int N, int C,
                               int groups, int act, float leaky_slope, int dtype, void* workspace, size_t ws_bytes,
                               void* stream) {
    YOLO_REQUIRE(x && gamma && beta && stats && dgamma && dbeta && workspace, "gn_act_bwd: null argument");
    if (int e = gn_check_shape(N, C, groups, act, leaky_slope, dtype, "gn_act_bwd")) return e;
    const int es = (int)elem_size(dtype);
    if (int e = gn_check_view(x, x, N, C, es, "gn_act_bwd", "x")) return e;
    if (int e = gn_check_view(dy, x, N, C, es, "gn_act_bwd", "dy")) return e;
    if (int e = gn_check_view(dx, x, N, C, es, "gn_act_bwd", "dx")) return e;
    YOLO_REQUIRE((uintptr_t)workspace % 16 == 0, "gn_act_bwd: workspace is not 16-byte aligned");
    if (ws_bytes < yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype))
        return fail(YOLO_E_WORKSPACE, "gn_act_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
                    yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype));
    GnParams p{};
    gn_shape(p, x, N, C, groups, es);
    p.x = gn_tensor(x, es);
    p.dy = gn_tensor(dy, es);
    p.y = gn_tensor(dx, es);
    p.gamma = gamma;
    p.beta = beta;
    p.stats = const_cast<float*>(stats);
    p.dgamma = dgamma;
    p.dbeta = dbeta;
    p.partial = workspace;
    p.sums = (float*)workspace + (size_t)N * p.chunks * 2 * C;
    p.terms = p.sums + (size_t)N * 2 * C;
    p.slope = leaky_slope;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid = gn_grid(p, es);
    GN_LAUNCH(gn_bwd_sums_kernel, grid, st, p);
    hipLaunchKernelGGL(gn_bwd_terms_kernel, dim3(groups, N), dim3(256), 0, st, p);
    GN_LAUNCH(gn_bwd_apply_kernel, grid, st, p);
    hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((2 * C + 255) / 256), dim3(256), 0, st, p);
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}
