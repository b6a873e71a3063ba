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
// Memory-bound: some twenty operations for each value of 2 or 4 bytes.  A pass reads or writes 16 bytes per lane.  Forward, sums are
// of differences from a pivot, fp32 over a thread's values (and a wave's, where a slab is in registers), fp64 from there on; backward
// they are fp32 within a workgroup.  Two forms, chosen by gn_whole_plan and gn_whole_first:
//   whole    a workgroup holds a slab (whole groups) of one image in registers: x and dy are read once, one launch
//   chunked  an image's slab over many workgroups, with a second pass over x and dy: sums, join, output (with few chunks the second
//            pass joins the sums itself: gn_split_joined)
// No atomics and a fixed order of additions: a call gives the same bits each time.
#include <type_traits>

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
    int slabs;             // whole-image kernels: slabs of an image
    int stream;            // the call moves more than the caches hold: loads and stores that do not stay in them
    int fold;              // whole-image kernel: channels folded in a thread (a power of two dividing Cg)
    const float* gamma;
    const float* beta;
    float* stats;          // [2][N][groups]: mean, r
    float* dgamma;
    float* dbeta;
    void* partial;         // forward: double [N][chunks][2][C]; backward: float [N][chunks][2][C]
    float* pivots;         // forward: [N][C], the values at pixel 0
    float* sums;           // backward: [N][2][C], one image's sums of d and of d * xh
    float* terms;          // backward: [2][N][groups], A and B
    float eps, slope;
    double inv_count;      // 1 / M
};

constexpr int GN_THREADS = 256;
constexpr int GN_MAX_CHUNKS = 256;

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

// K channels of a vector, the ones from part * K on.
template <typename E, int K>
__device__ __forceinline__ void gn_part(const u32x4& r, int part, float* v) {
    if constexpr (sizeof(E) == 2 && K == 4) {
        v[0] = __uint_as_float(r[2 * part] << 16);
        v[1] = __uint_as_float(r[2 * part] & 0xffff0000u);
        v[2] = __uint_as_float(r[2 * part + 1] << 16);
        v[3] = __uint_as_float(r[2 * part + 1] & 0xffff0000u);
    } else {
        GnVec<E>::unpack(r, v);
    }
}

// Byte offsets of a pixel's vector from the image's start in K tensors (below 2^31: the host checks), moved on by a fixed number
// of pixels without divisions or products.
template <int K>
struct GnCursor {
    int w, sw, W;
    int at[K], step[K], wrap[K];
    __device__ __forceinline__ GnCursor(int pixel, int pixels, int W_, int cb, const GnTensor* const (&t)[K]) : W(W_) {
        const int h = pixel / W, sh = pixels / W;
        w = pixel - h * W;
        sw = pixels - sh * W;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at[k] = h * t[k]->row + w * t[k]->pix + cb;
            step[k] = sh * t[k]->row + sw * t[k]->pix;
            wrap[k] = t[k]->row - W * t[k]->pix;
        }
    }
    __device__ __forceinline__ void next() {
        w += sw;
        const bool over = w >= W;
        w -= over ? W : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) at[k] += step[k] + (over ? wrap[k] : 0);
    }
};

// ST: a load of what is not read again soon, a store that leaves the caches to what is.  `base` is uniform, the offset a thread's.
template <int ST = 0>
__device__ __forceinline__ u32x4 gn_load(const char* base, unsigned at) {
    if constexpr (ST) return __builtin_nontemporal_load((const u32x4*)(base + at));
    return *(const u32x4*)(base + at);
}
template <int ST>
__device__ __forceinline__ void gn_store(char* base, unsigned at, const u32x4& v) {
    if constexpr (ST)
        __builtin_nontemporal_store(v, (u32x4*)(base + at));
    else
        *(u32x4*)(base + at) = v;
}
template <int N> struct GnCount { static constexpr int value = N; };
// f with the call's kind of loads and stores
template <typename F>
__device__ __forceinline__ void gn_with_stream(int stream, F f) {
    if (stream)
        f(GnCount<1>{});
    else
        f(GnCount<0>{});
}

constexpr int GN_LEAKY = YOLO_ACT_LEAKY, GN_SILU = YOLO_ACT_SILU;

// exp through v_exp_f32: the product with log2(e) is rounded before it, so that the error grows with t, about (|t| + 2) 2^-24 of the
// value, and 2^-23 more for the reciprocal: |t| below 10 where it counts.  t = -inf and +inf give 0 and 1.
__device__ __forceinline__ float gn_sigmoid(float t) { return __builtin_amdgcn_rcpf(1.f + __expf(-t)); }

template <int ACT>
__device__ __forceinline__ float gn_act(float t, float slope) {
    if constexpr (ACT == GN_SILU) return t * gn_sigmoid(t);
    return t > 0.f ? t : t * slope;
}

// d = dy * act'(t); `least` keeps the smallest |t| seen.  The leaky derivative jumps at t = 0 (slope at t == 0, torch's
// convention), and its side is decided exactly.  t = (x - mean) * (gamma r) + beta in fp32 is off by less than 2^-22 (|beta| +
// |t|): two roundings in each factor's product, which is about -beta where t is small, and one of the sum.  Where `least` ends
// up below 2^-20 times the largest |beta| of the channels (gn_near) -- one vector in some hundred thousand -- their values are
// done again with the sides from fp64 (gn_exact_side).
template <int ACT>
__device__ __forceinline__ float gn_act_grad(float dy, float t, float slope, float& least) {
    if constexpr (ACT == GN_SILU) {
        const float s = gn_sigmoid(t);
        return dy * (s * (1.f + t * (1.f - s)));
    } else {
        least = fminf(least, fabsf(t));
        return dy * (t > 0.f ? 1.f : slope);
    }
}
// 1 where t > 0 and slope elsewhere, from the channel's constants in LDS: {mean, r, gamma, beta}, `row` floats apart, at `c`.  The
// index is opaque and one call ends before the next one begins: the loops around the calls need the registers that constants
// loaded ahead would take.
__device__ __forceinline__ float gn_exact_side(float x, const float* lds, int c, int row, float slope) {
    asm volatile("" : "+v"(c));
    const double t = ((double)x - (double)lds[c]) * (double)lds[c + row] * (double)lds[c + 2 * row] + (double)lds[c + 3 * row];
    float side = t > 0.0 ? 1.f : slope;
    asm volatile("" : "+v"(side));
    return side;
}
template <int K>
__device__ __forceinline__ float gn_near(const float* beta) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < K; ++e) m = fmaxf(m, fabsf(beta[e]));
    return m * 0x1p-20f;
}

// The constants of a slab's channels in LDS: {mean, r, gamma, beta}, S floats each.
__device__ __forceinline__ void gn_stage(float* k, const GnParams& p, int n, int c0, int S) {
    for (int j = threadIdx.x; j < S && c0 + j < p.C; j += GN_THREADS) {
        const int g = (c0 + j) / p.Cg;
        k[j] = p.stats[n * p.groups + g];
        k[S + j] = p.stats[(p.N + n) * p.groups + g];
        k[2 * S + j] = p.gamma[c0 + j];
        k[3 * S + j] = p.beta[c0 + j];
    }
    __syncthreads();
}
// Makes the compiler forget what it has unpacked from the vectors, and loaded so far: kept between two passes it would not fit.
template <int NV>
__device__ __forceinline__ void gn_forget(u32x4 (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i])::"memory");
}

// What a thread needs of its V channels: t = (x - mean) * scale + beta with scale = gamma * r.
template <int V>
struct GnConst {
    float mean[V], scale[V], beta[V];
    __device__ __forceinline__ GnConst(const float* k, int S) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            mean[e] = k[e];
            scale[e] = k[2 * S + e] * k[S + e];
            beta[e] = k[3 * S + e];
        }
    }
};

// x - mean and d = dy * act'(t) of a vector's channels; k holds the constants of K of them, the ones from `part` * K on.
template <typename E, int ACT, int K>
__device__ __forceinline__ void gn_grads_of(const u32x4& x, const u32x4& dy, int part, const GnConst<K>& k, float near,
                                            const float* lds, int c, int row, float slope, float* xm, float* a) {
    float least = INFINITY;
    gn_part<E, K>(x, part, xm);
    gn_part<E, K>(dy, part, a);
#pragma unroll
    for (int e = 0; e < K; ++e) {
        xm[e] -= k.mean[e];
        a[e] = gn_act_grad<ACT>(a[e], fmaf(xm[e], k.scale[e], k.beta[e]), slope, least);
    }
    if (ACT == GN_LEAKY && __builtin_expect(least <= near, 0)) {
        u32x4 again[2] = {x, dy};
        gn_forget<2>(again);
        float v[K];
        gn_part<E, K>(again[0], part, v);
        gn_part<E, K>(again[1], part, a);
#pragma unroll
        for (int e = 0; e < K; ++e) a[e] *= gn_exact_side(v[e], lds, c + e, row, slope);
    }
}
template <typename E, int ACT>
__device__ __forceinline__ void gn_grads(const u32x4& x, const u32x4& dy, const GnConst<GnVec<E>::N>& k, float near, const float* lds, int c,
                                         int row, float slope, float* xm, float* a) {
    gn_grads_of<E, ACT, GnVec<E>::N>(x, dy, 0, k, near, lds, c, row, slope, xm, a);
}

// count steps, four at a time (their loads are all issued before the first is used), then one at a time.
template <typename F>
__device__ __forceinline__ void gn_in_fours(int count, F f) {
    int i = 0;
    for (; i + 4 <= count; i += 4) f(GnCount<4>{});
    for (; i < count; ++i) f(GnCount<1>{});
}

// count steps, U at a time: the loads of the next U are on their way while the last U are used.  load(r) takes the next step's
// vectors, use(r) uses them.
template <int U, int K, typename L, typename F>
__device__ __forceinline__ void gn_pipelined(int count, L load, F use) {
    u32x4 now[U][K];
    int i = 0;
    if (count >= U) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(now[u]);
        for (i = U; i + U <= count; i += U) {
            u32x4 next[U][K];
#pragma unroll
            for (int u = 0; u < U; ++u) load(next[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) use(now[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < K; ++k) now[u][k] = next[u][k];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) use(now[u]);
    }
    for (; i < count; ++i) {
        load(now[0]);
        use(now[0]);
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
// partial[n][chunk][0 / 1][c] = sum of x - P, of its square over the chunk's pixels, P the channel's value at pixel 0.  A thread sums
// differences from the first value it sees (fp32; the values of a few dozen pixels differ from it by about their spread), and goes over
// to fp64 and to P after that: squares about zero would leave the variance of a group that is constant at 1000 off by 1e-4 of eps
// even in fp64.
// Bound by the read: 64 x 208 x 208 x 64 bf16, 354 MB in 65 us, 5.4 TB/s.  256 threads, at most 128 pixels to a thread: 2048
// workgroups, so that a CU has the loads of several in flight.
template <typename E>
__global__ void __launch_bounds__(GN_THREADS, 5) gn_sums_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ double red[GN_THREADS * V];
    __shared__ u32x4 origin[GN_THREADS];  // pixel 0's vector, which needs no registers here during the loop
    const GnLane l = gn_lane<E>(p);
    const int n = blockIdx.z, first = blockIdx.x * p.chunk, last = min(first + p.chunk, p.HW);
    const char* base = p.x.p + n * p.x.img;
    const int cb = l.c * (int)sizeof(E);
    float k[V], s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
    int count = 0;
    const u32x4 pixel0 = gn_load(base, l.on ? cb : 0);
    if (l.on && first + l.pl < last) {
        GnCursor<1> c(first + l.pl, p.PL, p.W, cb, {&p.x});
        count = (last - first - l.pl + p.PL - 1) / p.PL;
        GnVec<E>::unpack(gn_load(base, c.at[0]), k);
        origin[threadIdx.x] = pixel0;
        c.next();
        gn_pipelined<4, 1>(
            count - 1,
            [&](u32x4* r) {
                r[0] = gn_load(base, c.at[0]);
                c.next();
            },
            [&](const u32x4* r) {
                float v[V];
                GnVec<E>::unpack(r[0], v);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = v[e] - k[e];
                    s[e] += d;
                    q[e] = fmaf(d, d, q[e]);
                }
            });
    }
    const int S = p.VS * V;
    float from[V] = {};
    if (count) GnVec<E>::unpack(origin[threadIdx.x], from);
    if (blockIdx.x == 0 && l.on && l.pl == 0)
#pragma unroll
        for (int e = 0; e < V; ++e) p.pivots[(long long)n * p.C + l.c + e] = from[e];
    double* out = (double*)p.partial + (((long long)n * p.chunks + blockIdx.x) * 2) * p.C + blockIdx.y * S;
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double K = (double)k[e] - (double)from[e], sd = s[e];
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

// sum[k] += value k of the rows from, from + step, ... below count, U rows' loads at a time, the last ones too: each row is a trip to
// memory of 1 us.  load(row, k) is called with rows below count only.
template <int U, int K, typename P, typename L>
__device__ __forceinline__ void gn_sum_rows(int from, int count, int step, double (&sum)[K], L load) {
    for (int i = from; i < count; i += U * step) {
        P v[U][K];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                v[u][k] = 0;
                if (i + u * step < count) v[u][k] = load(i + u * step, k);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < K; ++k) sum[k] += (double)v[u][k];
    }
}
// The sums of x - P and its square over an image's channel -> about P - by
__device__ __forceinline__ void gn_move_origin(const GnParams& p, double by, double& sum, double& square) {
    square += by * (2.0 * sum + p.HW * by);
    sum += p.HW * by;
}
__device__ __forceinline__ float gn_rstd(const GnParams& p, double var) {
    return (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)p.eps));
}

// The chunks' sums of the groups of about 64 channels of one image, in fp64 and in the chunks' order: lanes are channels, the
// sixteen waves take the chunks in turn.  Forward: mean and r of a group.  Backward: the image's sums of each channel, and the
// group's two terms from gamma times them.  Latency-bound, 4 to 5 us.
constexpr int GN_JOIN = 16;
template <bool BWD>
__global__ void __launch_bounds__(GN_JOIN * 64) gn_join_kernel(const GnParams p) {
    typedef typename std::conditional<BWD, float, double>::type P;
    __shared__ double red[2][GN_JOIN][64];
    const int col = threadIdx.x & 63, row = threadIdx.x >> 6, n = blockIdx.y;
    const int per = p.Cg < 64 ? 64 / p.Cg : 1, g0 = blockIdx.x * per, groups = min(per, p.groups - g0), width = groups * p.Cg;
    const P* part = (const P*)p.partial + (long long)n * p.chunks * 2 * p.C + g0 * p.Cg;
    double A = 0.0, B = 0.0;
    for (int c0 = 0; c0 < width; c0 += 64) {
        const int c = c0 + col;
        double sum[2] = {0.0, 0.0};
        if (c < width)
            gn_sum_rows<8, 2, P>(row, p.chunks, GN_JOIN, sum, [&](int i, int k) { return part[((long long)i * 2 + k) * p.C + c]; });
        double a = sum[0], b = sum[1];
        red[0][row][col] = a;
        red[1][row][col] = b;
        __syncthreads();
        if (row == 0) {
            for (int w = 1; w < GN_JOIN; ++w) {
                a += red[0][w][col];
                b += red[1][w][col];
            }
            if (!BWD && c < width) {  // about the group's pivot, its first channel's
                const float* P = p.pivots + (long long)n * p.C + g0 * p.Cg;
                gn_move_origin(p, (double)P[c] - (double)P[c / p.Cg * p.Cg], a, b);
            }
            if (BWD && c < width) {
                p.sums[((long long)n * 2) * p.C + g0 * p.Cg + c] = (float)a;
                p.sums[((long long)n * 2 + 1) * p.C + g0 * p.Cg + c] = (float)b;
                const double gamma = p.gamma[g0 * p.Cg + c];
                a *= gamma;
                b *= gamma;
            }
            red[0][0][col] = a;
            red[1][0][col] = b;
        }
        __syncthreads();
        if ((int)threadIdx.x < groups) {  // groups > 1: all their channels are here; else the next 64 of the one group
            const int first = groups > 1 ? threadIdx.x * p.Cg : 0, last = groups > 1 ? first + p.Cg : min(64, width - c0);
            for (int i = first; i < last; ++i) {
                A += red[0][0][i];
                B += red[1][0][i];
            }
        }
        __syncthreads();
    }
    if ((int)threadIdx.x >= groups) return;
    const int g = n * p.groups + g0 + threadIdx.x;
    if (BWD) {
        p.terms[g] = (float)(A * p.inv_count);
        p.terms[p.N * p.groups + g] = (float)(B * p.inv_count);
    } else {
        const double d = A * p.inv_count;
        p.stats[g] = (float)((double)p.pivots[(long long)n * p.C + (g0 + threadIdx.x) * p.Cg] + d);
        p.stats[p.N * p.groups + g] = gn_rstd(p, B * p.inv_count - d * d);
    }
}

// The same for the `width` channels of a slab (whole groups) from c0 on, by a workgroup that goes on with them: the group sums of its
// groups, handed to done(group in the slab, sum, sum, lane) in 16 lanes each.  16 bytes of sums a lane; `red` has room for a workgroup's.
template <bool BWD, typename F>
__device__ __forceinline__ void gn_join_slab(const GnParams& p, int n, int c0, int width, double* red, F done) {
    typedef typename std::conditional<BWD, float, double>::type P;
    constexpr int K = 16 / (int)sizeof(P);  // channels of a lane; width and c0 are multiples of it
    typedef P PK __attribute__((ext_vector_type(K)));
    const int lanes = width / K, rows = min(GN_THREADS / lanes, p.chunks), row = threadIdx.x / lanes, col = (threadIdx.x - row * lanes) * K;
    const P* part = (const P*)p.partial + (long long)n * p.chunks * 2 * p.C + c0 + col;
    double by = 0.0;  // forward: from the channel's pivot to the group's
    if (!BWD && (int)threadIdx.x < width) {
        const float* pivot = p.pivots + (long long)n * p.C + c0;
        by = (double)pivot[threadIdx.x] - (double)pivot[threadIdx.x / p.Cg * p.Cg];
    }
    double sum[2][K];
#pragma unroll
    for (int k = 0; k < K; ++k) sum[0][k] = sum[1][k] = 0.0;
    constexpr int U = 4;  // rows' loads at a time, the last ones too: each is a trip to memory
    if (row < rows)
        for (int i = row; i < p.chunks; i += U * rows) {
            PK v[U][2];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    v[u][w] = PK(0);
                    if (i + u * rows < p.chunks) v[u][w] = *(const PK*)(part + ((long long)(i + u * rows) * 2 + w) * p.C);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < K; ++k) sum[w][k] += (double)v[u][w][k];
        }
    double total[2] = {0.0, 0.0};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (row < rows)
#pragma unroll
            for (int k = 0; k < K; ++k) red[row * width + col + k] = sum[w][k];
        __syncthreads();
        if ((int)threadIdx.x < width)
            for (int r = 0; r < rows; ++r) total[w] += red[r * width + threadIdx.x];
        __syncthreads();
    }
    if ((int)threadIdx.x < width) {
        const double gamma = BWD ? p.gamma[c0 + threadIdx.x] : 1.f;
        if constexpr (!BWD) gn_move_origin(p, by, total[0], total[1]);
        red[threadIdx.x] = gamma * total[0];
        red[GN_THREADS + threadIdx.x] = gamma * total[1];
    }
    __syncthreads();
    const int sub = threadIdx.x & 15, groups = width / p.Cg;
    for (int g0 = 0; g0 < groups; g0 += GN_THREADS / 16) {
        const int g = g0 + (threadIdx.x >> 4);
        double A = 0.0, B = 0.0;
        if (g < groups)
            for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) {
                A += red[i];
                B += red[GN_THREADS + i];
            }
        for (int o = 8; o; o >>= 1) {
            A += __shfl_xor(A, o);
            B += __shfl_xor(B, o);
        }
        if (g < groups) done(g, A, B, sub);
    }
    __syncthreads();
}
// ------------------------------------------------------------------------------------------------ forward, output
// y = act((x - mean) * (gamma r) + beta) [+ residual], images and chunks in the reverse order of the sums: what was read last is
// still in the cache in front of HBM.  64 x 208 x 208 x 64 bf16: 709 MB in 123 us, 5.8 TB/s.  (x * (gamma r) + (beta - mean gamma r), an
// operation less, would round mean gamma r: in a nearly constant group of mean 1000 that is 1e-2, in bf16 too more than the output's
// own rounding.)
template <typename E, int ACT, bool JOIN = false>
__global__ void __launch_bounds__(GN_THREADS, JOIN ? 6 : 8) gn_apply_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ double red[JOIN ? 2 * GN_THREADS : 1];
    __shared__ float of[2][JOIN ? GN_THREADS : 1];
    const GnLane l = gn_lane<E>(p);
    // the pass before this one walked forwards: its last chunks are the ones still in the caches
    const int n = p.N - 1 - blockIdx.z, chunk = p.chunks - 1 - blockIdx.x;
    const int first = chunk * p.chunk, last = min(first + p.chunk, p.HW), c0 = blockIdx.y * p.VS * V;
    if constexpr (JOIN)
        gn_join_slab<false>(p, n, c0, min(p.VS * V, p.C - c0), red, [&](int g, double A, double B, int sub) {
            const double d = A * p.inv_count;
            const float mean = (float)((double)p.pivots[(long long)n * p.C + c0 + g * p.Cg] + d), r = gn_rstd(p, B * p.inv_count - d * d);
            for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) {
                of[0][i] = mean;
                of[1][i] = r;
            }
            if (sub == 0 && chunk == 0) {
                p.stats[n * p.groups + c0 / p.Cg + g] = mean;
                p.stats[(p.N + n) * p.groups + c0 / p.Cg + g] = r;
            }
        });
    if (!l.on || first + l.pl >= last) return;
    float mean[V], scale[V], beta[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (l.c + e) / p.Cg;
        mean[e] = JOIN ? of[0][l.c - c0 + e] : p.stats[n * p.groups + g];
        scale[e] = p.gamma[l.c + e] * (JOIN ? of[1][l.c - c0 + e] : p.stats[(p.N + n) * p.groups + g]);
        beta[e] = p.beta[l.c + e];
    }
    const int cb = l.c * (int)sizeof(E);
    const char* x = p.x.p + n * p.x.img;
    char* y = p.y.p + n * p.y.img;
    const int count = (last - first - l.pl + p.PL - 1) / p.PL;
    gn_with_stream(p.stream, [&](auto st) {
        constexpr int ST = decltype(st)::value;
        auto put = [&](const u32x4& raw, const u32x4* res, unsigned to) {
            float v[V];
            GnVec<E>::unpack(raw, v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = gn_act<ACT>(fmaf(v[e] - mean[e], scale[e], beta[e]), p.slope);
            if (res) {
                float a[V];
                GnVec<E>::unpack(*res, a);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += a[e];
            }
            gn_store<ST>(y, to, GnVec<E>::pack(v));
        };
        if (p.r.p) {
            const char* r = p.r.p + n * p.r.img;
            GnCursor<3> c(first + l.pl, p.PL, p.W, cb, {&p.x, &p.r, &p.y});
#pragma unroll 4
            for (int i = 0; i < count; ++i) {
                const u32x4 res = gn_load<ST>(r, c.at[1]);
                put(gn_load<ST>(x, c.at[0]), &res, c.at[2]);
                c.next();
            }
        } else {
            GnCursor<2> c(first + l.pl, p.PL, p.W, cb, {&p.x, &p.y});
#pragma unroll 4
            for (int i = 0; i < count; ++i) {
                put(gn_load<ST>(x, c.at[0]), nullptr, c.at[1]);
                c.next();
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ backward, sums
// partial[n][chunk][0 / 1][c] = sum of d, of d * xh over the chunk's pixels, two pairs of vectors ahead.  64 x 208 x 208 x
// 64 bf16: 709 MB in 118 us, 6.0 TB/s.
template <typename E, int ACT>
__global__ void __launch_bounds__(GN_THREADS, 4) gn_bwd_sums_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ __attribute__((aligned(16))) float lds[4 * GN_THREADS * V];  // the slab's constants, then its threads' sums
    const GnLane l = gn_lane<E>(p);
    const int n = blockIdx.z, first = blockIdx.x * p.chunk, last = min(first + p.chunk, p.HW), S = p.VS * V;
    const float* mine = lds + (l.c - blockIdx.y * S);
    gn_stage(lds, p, n, blockIdx.y * S, S);
    float sd[V], sx[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sd[e] = sx[e] = 0.f;
    if (l.on && first + l.pl < last) {
        const GnConst<V> k(mine, S);
        const int cb = l.c * (int)sizeof(E);
        const char* x = p.x.p + n * p.x.img;
        const char* dy = p.dy.p + n * p.dy.img;
        const int count = (last - first - l.pl + p.PL - 1) / p.PL;
        const float near = gn_near<V>(k.beta);
        GnCursor<2> c(first + l.pl, p.PL, p.W, cb, {&p.x, &p.dy});
        gn_pipelined<2, 2>(
            count,
            [&](u32x4* r) {
                r[0] = gn_load(x, c.at[0]);
                r[1] = gn_load(dy, c.at[1]);
                c.next();
            },
            [&](const u32x4* r) {
                float xm[V], a[V];
                gn_grads<E, ACT>(r[0], r[1], k, near, lds, l.c - blockIdx.y * S, S, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sd[e] += a[e];
                    sx[e] = fmaf(a[e], xm[e], sx[e]);
                }
            });
    }
    __syncthreads();
    float* red = lds;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        red[threadIdx.x * V + e] = sd[e];
        red[(GN_THREADS + threadIdx.x) * V + e] = sx[e];
    }
    __syncthreads();
    float* out = (float*)p.partial + (((long long)n * p.chunks + blockIdx.x) * 2) * p.C + blockIdx.y * S;
    for (int j = threadIdx.x; j < S && blockIdx.y * S + j < p.C; j += GN_THREADS) {
        float a = 0.f, b = 0.f;
        for (int i = 0; i < p.PL; ++i) {
            a += red[i * S + j];
            b += red[GN_THREADS * V + i * S + j];
        }
        out[j] = a;
        out[p.C + j] = b * p.stats[(p.N + n) * p.groups + (blockIdx.y * S + j) / p.Cg];
    }
}

// dgamma, dbeta: the images' sums.  A workgroup has 32 of the 2 C columns (d sums, then d * xh sums), the i-th such set of them,
// and eight rows at a time.
__device__ __forceinline__ void gn_params(const GnParams& p, int set, double (*red)[32], const float* sums, int rows) {
    const int col = threadIdx.x & 31, row = threadIdx.x >> 5, i = set * 32 + col;
    double sum[1] = {0.0};
    if (i < 2 * p.C) gn_sum_rows<8, 1, float>(row, rows, 8, sum, [&](int n, int) { return sums[(long long)n * 2 * p.C + i]; });
    double a = sum[0];
    red[row][col] = a;
    __syncthreads();
    if (row == 0 && i < 2 * p.C) {
        for (int k = 1; k < 8; ++k) a += red[k][col];
        if (i < p.C)
            p.dbeta[i] = (float)a;
        else
            p.dgamma[i - p.C] = (float)a;
    }
    __syncthreads();
}
__global__ void __launch_bounds__(GN_THREADS) gn_bwd_params_kernel(const GnParams p) {
    __shared__ double red[8][32];
    gn_params(p, blockIdx.x, red, p.sums, p.N);
}

// ------------------------------------------------------------------------------------------------ backward, output
// dx = d * scale - (x - mean) * (r r B) - r A, four pixels at a time, images and chunks in the reverse order of the sums (64 x
// 208 x 208 x 64 bf16: 1063 MB in 178 us, 6.0 TB/s).  The first plane of the grid sums dgamma and dbeta: a launch
// of its own for them is 3 us.
template <typename E, int ACT, bool JOIN = false>
__global__ void __launch_bounds__(GN_THREADS, 4) gn_bwd_apply_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    __shared__ __attribute__((aligned(16))) float lds[4 * GN_THREADS * V];
    if (blockIdx.z == 0) {
        for (int set = blockIdx.y * p.chunks + blockIdx.x; set * 32 < 2 * p.C; set += p.chunks * gridDim.y)
            gn_params(p, set, (double (*)[32])lds, JOIN ? (const float*)p.partial : p.sums, JOIN ? p.N * p.chunks : p.N);
        return;
    }
    const GnLane l = gn_lane<E>(p);
    const int n = p.N - blockIdx.z, chunk = p.chunks - 1 - blockIdx.x, S = p.VS * V;
    const int first = chunk * p.chunk, last = min(first + p.chunk, p.HW);
    const float* mine = lds + (l.c - blockIdx.y * S);
    gn_stage(lds, p, n, blockIdx.y * S, S);
    float* terms = lds + 4 * GN_THREADS;  // JOIN: behind the constants of at most GN_THREADS channels; then the sums to join
    if constexpr (JOIN)
        gn_join_slab<true>(p, n, blockIdx.y * S, min(S, p.C - (int)blockIdx.y * S), (double*)(lds + 6 * GN_THREADS),
                           [&](int g, double A, double B, int sub) {
                               for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) {
                                   terms[i] = (float)(A * p.inv_count);
                                   terms[GN_THREADS + i] = (float)(B * p.inv_count);
                               }
                           });
    if (!l.on || first + l.pl >= last) return;
    const GnConst<V> k(mine, S);
    float k0[V], k1[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = (l.c + e) / p.Cg, c = l.c + e - blockIdx.y * S;
        const float r = p.stats[(p.N + n) * p.groups + g];
        k0[e] = -r * (JOIN ? terms[c] : p.terms[n * p.groups + g]);
        k1[e] = -r * r * (JOIN ? terms[GN_THREADS + c] : p.terms[(p.N + n) * p.groups + g]);
    }
    const float near = gn_near<V>(k.beta);
    const int cb = l.c * (int)sizeof(E);
    const char* x = p.x.p + n * p.x.img;
    const char* dy = p.dy.p + n * p.dy.img;
    char* y = p.y.p + n * p.y.img;
    const int count = (last - first - l.pl + p.PL - 1) / p.PL;
    gn_with_stream(p.stream, [&](auto st) {
        constexpr int ST = decltype(st)::value;
        GnCursor<2> c(first + l.pl, p.PL, p.W, cb, {&p.x, &p.dy});
        GnCursor<1> cy(first + l.pl, p.PL, p.W, cb, {&p.y});
        gn_in_fours(count, [&](auto u) {
            constexpr int U = decltype(u)::value;
            u32x4 vr[U], dr[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                vr[i] = gn_load<ST>(x, c.at[0]);
                dr[i] = gn_load<ST>(dy, c.at[1]);
                c.next();
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float xm[V], a[V];
                gn_grads<E, ACT>(vr[i], dr[i], k, near, lds, l.c - blockIdx.y * S, S, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < V; ++e) a[e] = fmaf(a[e], k.scale[e], fmaf(xm[e], k1[e], k0[e]));
                gn_store<ST>(y, cy.at[0], GnVec<E>::pack(a));
                cy.next();
            }
        });
    });
}

// ------------------------------------------------------------------------------------------------ whole images
// One workgroup holds all pixels of a slab of whole groups of one image in registers, so that x (and dy) are read once: VS
// vectors of 16 bytes per pixel, 64 / VS pixels next to each other in a wave, NV vectors to a thread.  The statistics are then
// the two sums of the definition (mean, then squares about it), fp32 in a thread, over its channels of a group and over its wave's pixel
// lanes (at most 22 + 3 + 6 additions in a row), fp64 between waves.  The first sum is of differences from the channel's value at pixel 0:
// raw values far from zero would lose the mean's last digits, and a nearly constant group (r up to 1 / sqrt(eps)) its output's first
// ones.  64 x 52 x 52 x 256 bf16 with a residual: 266 MB in 58 us, 4.6 TB/s (one round of 256 workgroups that load, add up and store at
// the same time); one image of 13 x 13 x 1024: 6.8 us, of which a launch and the way to memory and back are most.
constexpr int GN_SLAB = 128;  // most channels of a slab (at most the threads of the smallest workgroup)
constexpr int GN_WAVES = 16;

struct GnSeat {
    int slab, n;
    int wave, waves, pl, c, cs, first, step, count;  // c: channel; cs: channel in the slab; pixels first + i * step, i < count
    int full, most;  // every lane has steps i < full, no lane has i >= most; most is full or full + 1
    bool on;
};
template <typename E>
__device__ __forceinline__ GnSeat gn_seat(const GnParams& p) {
    GnSeat s;
    // consecutive workgroups go to the eight XCDs in turn: each XCD gets a run of neighbouring slabs, so that slabs that share a
    // cache line are read through one L2 at about the same time
    const int total = p.slabs * p.N, q = total >> 3, rest = total & 7, xcd = blockIdx.x & 7;
    const int at = xcd * q + min(xcd, rest) + (blockIdx.x >> 3);
    s.n = at / p.slabs;
    s.slab = at - s.n * p.slabs;
    const int lane = threadIdx.x & 63;
    s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    s.waves = blockDim.x >> 6;
    s.step = s.waves * p.PL;
    s.full = p.HW / s.step;
    s.most = (p.HW + s.step - 1) / s.step;
    s.pl = lane / p.VS;
    s.cs = (lane - s.pl * p.VS) * GnVec<E>::N;
    s.c = s.slab * p.VS * GnVec<E>::N + s.cs;
    s.on = s.pl < p.PL && s.c < p.C;
    s.first = s.wave * p.PL + s.pl;
    s.count = s.on && s.first < p.HW ? (p.HW - s.first + s.step - 1) / s.step : 0;
    return s;
}
// The thread's vectors of K tensors; where it has none a load takes pixel 0's, so that all of them are plain loads inside the view,
// issued one after the other.
template <int K>
struct GnWalk {
    GnCursor<K> c;
    int at0;
    __device__ __forceinline__ GnWalk(const GnParams& p, const GnSeat& s, int cb, const GnTensor* const (&t)[K])
        : c(s.count ? s.first : 0, s.step, p.W, cb, t), at0(cb) {}
    template <int ST, bool ALL>
    __device__ __forceinline__ u32x4 load(int k, int i, const GnSeat& s, const char* base) const {
        return gn_load<ST>(base, ALL || i < s.count ? c.at[k] : at0);
    }
};
// ... and zeros there
template <int NV>
__device__ __forceinline__ void gn_blank(u32x4 (&v)[NV], const GnSeat& s) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (i >= s.full && i >= s.count) v[i] = u32x4{0u, 0u, 0u, 0u};
}

template <typename E>
__device__ __forceinline__ void gn_put_four(u32x4& r, int h, const float* v) {
    if constexpr (sizeof(E) == 2) {
        r[2 * h] = pack_bf16x2(v[0], v[1]);
        r[2 * h + 1] = pack_bf16x2(v[2], v[3]);
    } else {
        r = GnVec<float>::pack(v);
    }
}

// A cursor over the thread's pixels whose positions the compiler does not keep from an earlier walk.
template <int K>
__device__ __forceinline__ GnCursor<K> gn_again(const GnParams& p, const GnSeat& s, int cb, const GnTensor* const (&t)[K]) {
    int first = s.first;
    asm volatile("" : "+v"(first));
    return GnCursor<K>(first, s.step, p.W, cb, t);
}

// The sum over a wave's pixel lanes, valid in those of pixel lane 0.
template <typename T>
__device__ __forceinline__ T gn_over_pixels(T v, const GnParams& p, int pl, int top) {
    for (int o = top; o; o >>= 1) {
        const T w = __shfl_down(v, o * p.VS);
        v += pl + o < p.PL ? w : T(0);
    }
    return v;
}

// part[wave][cell] <- sums of the slab's cells (fold channels each) over the wave's pixels; then the group sums, handed to
// done(group in the slab, sum, lane) in 16 lanes each.
template <int V, typename T, typename F>
__device__ __forceinline__ void gn_group_sums(T (&s)[V], T (*part)[GN_SLAB], const GnParams& p, const GnSeat& t, int groups,
                                              int top, F done) {
    if (p.fold >= 2)
#pragma unroll
        for (int e = 0; e < V; e += 2) s[e] += s[e + 1];
    if (p.fold >= 4)
#pragma unroll
        for (int e = 0; e < V; e += 4) s[e] += s[e + 2];
    if constexpr (V == 8)
        if (p.fold >= 8) s[0] += s[4];
#pragma unroll
    for (int e = 0; e < V; ++e)
        if ((e & (p.fold - 1)) == 0) {
            const T v = gn_over_pixels(s[e], p, t.pl, top);
            if (t.pl == 0 && t.on) part[t.wave][(t.cs + e) / p.fold] = v;
        }
    __syncthreads();
    const int cells = p.Cg / p.fold, items = cells * t.waves, sub = threadIdx.x & 15;  // 16 lanes to a group
    for (int g0 = 0; g0 < groups; g0 += blockDim.x >> 4) {
        const int g = g0 + (threadIdx.x >> 4);
        double a = 0.0;
        if (g < groups)
            for (int i = sub; i < items; i += 16) {
                const int w = i / cells;
                a += (double)part[w][g * cells + i - w * cells];
            }
        for (int o = 8; o; o >>= 1) a += __shfl_xor(a, o);
        if (g < groups) done(g, a, sub);
    }
    __syncthreads();
}

__device__ __forceinline__ int gn_top(int pl) {  // the first distance of a tree over pl lanes
    int o = 1;
    while (o < pl) o <<= 1;
    return o >> 1;
}

//
// TALL: slabs that do not fit.  A thread's first NV vectors are in registers, the next GN_KEPT_FWD in LDS, and what is left is read
// again; those beyond NV are summed first, as in gn_sums_kernel (pivots; fp64 sums of differences and squares), the others by the
// definition.  64 x 60 x 60 x 256 bf16 with a residual: 78 us, with 64 B whole 98; without one 51 and 67.  Twelve vectors in
// registers leave room for the residual's (with 14 and 16 that call took 5 and 7 us longer than with 12, the one without as long).
constexpr int GN_KEPT_FWD = 8;
enum { GN_WHOLE, GN_TALL, GN_TALL_RESIDUAL };
template <typename E, int ACT, int NV, int FORM = GN_WHOLE>
__global__ void __launch_bounds__(1024) gn_whole_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N;
    constexpr bool TALL = FORM != GN_WHOLE;
    __shared__ double parts[TALL ? GN_WAVES : GN_WAVES / 2][GN_SLAB];
    __shared__ u32x4 kept[TALL ? GN_KEPT_FWD : 1][TALL ? 1024 : 1];
    // by group: the sums of x - P and of its square over what is not in registers, P the pivot of the group's first channel
    __shared__ double others[2][TALL ? GN_SLAB : 1];
    float (*part)[GN_SLAB] = (float (*)[GN_SLAB])parts;
    __shared__ __attribute__((aligned(16))) float mean_of[GN_SLAB], scale_of[GN_SLAB], beta_of[GN_SLAB];  // by channel
    __shared__ double off_of[GN_SLAB];  // by group: the mean minus its fp32 value
    __shared__ float pivot_of[GN_SLAB];  // by channel: pixel 0's value
    const GnSeat t = gn_seat<E>(p);
    const int n = t.n, S = p.VS * V, c0 = t.slab * S, g0 = c0 / p.Cg, top = gn_top(p.PL), width = min(S, p.C - c0);
    const int groups = width / p.Cg;
    const int cb = (t.on ? t.c : 0) * (int)sizeof(E);
    const int mine = min((int)threadIdx.x, width - 1);  // width <= GN_SLAB <= threads; these two loads come back first
    const float gamma = p.gamma[c0 + mine], beta = p.beta[c0 + mine];
    const char* x = p.x.p + n * p.x.img;
    const int more = TALL ? max(t.count - NV, 0) : 0;
    // sums in registers are of differences from pixel 0's values (its vector is also what a thread has where it has no pixel)
    const u32x4 pivot = gn_load(x, cb);
    auto share_pivot = [&] {
        float k0[V];
        GnVec<E>::unpack(pivot, k0);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (t.on && t.first == 0) pivot_of[t.cs + e] = k0[e];
    };
    if constexpr (TALL) {  // sums of differences from the thread's first value, as gn_sums_kernel
        float k[V], s[V], q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
        if (more) {
            GnCursor<1> c(t.first + NV * t.step, t.step, p.W, cb, {&p.x});
            const u32x4 r0 = gn_load(x, c.at[0]);
            c.next();
            kept[0][threadIdx.x] = r0;
            GnVec<E>::unpack(r0, k);
            int i = 1;
            gn_pipelined<4, 1>(
                more - 1,
                [&](u32x4* r) {
                    r[0] = gn_load(x, c.at[0]);
                    c.next();
                },
                [&](const u32x4* r) {
                    if (i < GN_KEPT_FWD) kept[i][threadIdx.x] = r[0];
                    ++i;
                    float f[V];
                    GnVec<E>::unpack(r[0], f);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float d = f[e] - k[e];
                        s[e] += d;
                        q[e] = fmaf(d, d, q[e]);
                    }
                });
        }
        share_pivot();
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            double m[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double K = (double)k[e] - (double)pivot_of[(t.cs + e) / p.Cg * p.Cg], sd = s[e];
                m[e] = which == 0 ? more * K + sd : (double)q[e] + K * (2.0 * sd + more * K);
            }
            gn_group_sums<V>(m, parts, p, t, groups, top, [&](int g, double sum, int sub) {
                if (sub == 0) others[which][g] = sum;
            });
        }
    }
    u32x4 v[NV];
    gn_with_stream(p.stream, [&](auto st) {
        GnWalk<1> walk(p, t, cb, {&p.x});
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = walk.template load<decltype(st)::value, TALL>(0, i, t, x);
            walk.c.next();
        }
    });
    if constexpr (!TALL) share_pivot();
    float s[V], k0[V];
    GnVec<E>::unpack(pivot, k0);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (TALL || i < t.most) {
            float f[V];
            GnVec<E>::unpack(v[i], f);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += f[e] - k0[e];
        }
    gn_group_sums<V>(s, part, p, t, groups, top, [&](int g, double sum, int sub) {
        const double P = pivot_of[g * p.Cg];
        double at = 0.0;
        for (int i = sub; i < p.Cg; i += 16) at += (double)pivot_of[g * p.Cg + i] - P;
        for (int o = 8; o; o >>= 1) at += __shfl_xor(at, o);
        sum += at * (TALL ? NV * t.step : p.HW);
        const double mean = P + (TALL ? sum + others[0][g] : sum) * p.inv_count;
        for (int i = sub; i < p.Cg; i += 16) mean_of[g * p.Cg + i] = (float)mean;
        if (sub == 0) {
            off_of[g] = mean - (double)(float)mean;
            p.stats[n * p.groups + g0 + g] = (float)mean;
        }
    });
    gn_forget<NV>(v);
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {  // four channels at a time: the registers are full
        if (h) gn_forget<NV>(v);
        float mean[4], q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) mean[e] = mean_of[t.cs + 4 * h + e];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (TALL || i < t.full || i < t.count) {
                float f[4];
                gn_part<E, 4>(v[i], h, f);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float d = f[e] - mean[e];
                    q[e] = fmaf(d, d, q[e]);
                }
            }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * h + e] = q[e];
    }
    gn_group_sums<V>(s, part, p, t, groups, top, [&](int g, double sum, int sub) {
        if constexpr (TALL) {
            const double m = (double)mean_of[g * p.Cg] - (double)pivot_of[g * p.Cg], count = (double)(p.HW - NV * t.step) * p.Cg;
            sum += others[1][g] + m * (m * count - 2.0 * others[0][g]);
        }
        const double off = off_of[g], var = sum * p.inv_count - off * off;
        const float r = gn_rstd(p, var);
        for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) scale_of[i] = r;
        if (sub == 0) p.stats[(p.N + n) * p.groups + g0 + g] = r;
    });
    if ((int)threadIdx.x < width) {
        scale_of[threadIdx.x] *= gamma;
        beta_of[threadIdx.x] = beta;
    }
    __syncthreads();
    if (!t.count) return;
    gn_forget<NV>(v);
    const bool residual = TALL ? FORM == GN_TALL_RESIDUAL : p.r.p != nullptr;
    const char* res = p.r.p + n * p.r.img;  // read where there is one
    char* y = p.y.p + n * p.y.img;
    // Where there are no registers for the constants they come from LDS, for four channels of a vector at a time: 64 x 40 x 40 x 256, 16
    // vectors, with a residual 39.4 -> 37.8 us; 64 x 60 x 60 x 256, tall, with one 80.8 -> 78.0, without one 51.8 and 54.6.
    constexpr bool KEEP = NV < 16 && FORM != GN_TALL_RESIDUAL;
    constexpr int K = KEEP ? V : 4;
    float mean[K], scale[K], bias[K];
    auto constants = [&](int cs) {
#pragma unroll
        for (int e = 0; e < K; ++e) {
            mean[e] = mean_of[cs + e];
            scale[e] = scale_of[cs + e];
            bias[e] = beta_of[cs + e];
        }
    };
    if (KEEP) constants(t.cs);
    gn_with_stream(p.stream, [&](auto st) {
        constexpr int ST = decltype(st)::value;
        auto put = [&](const u32x4& raw, const u32x4* r, unsigned to) {
            u32x4 out;
#pragma unroll
            for (int h = 0; h < V / K; ++h) {
                if constexpr (!KEEP) {
                    int cs = t.cs + h * K;
                    asm volatile("" : "+v"(cs));
                    constants(cs);
                }
                float f[K];
                gn_part<E, K>(raw, h, f);
#pragma unroll
                for (int e = 0; e < K; ++e) f[e] = gn_act<ACT>(fmaf(f[e] - mean[e], scale[e], bias[e]), p.slope);
                if (r) {
                    float a[K];
                    gn_part<E, K>(*r, h, a);
#pragma unroll
                    for (int e = 0; e < K; ++e) f[e] += a[e];
                }
                if constexpr (KEEP)
                    out = GnVec<E>::pack(f);
                else
                    gn_put_four<E>(out, h, f);
            }
            gn_store<ST>(y, to, out);
        };
        if (residual) {  // the residual of the next vectors is on its way while the last ones are finished
            // above 16 vectors more would not stay in registers (64 x 52 x 52 x 256: 57.7 us with 1, 60.4 with 2, 65.7 with 4)
            constexpr int AHEAD = NV > 16 ? 1 : 4;
            GnWalk<1> ahead(p, t, cb, {&p.r});
            GnCursor<1> c = gn_again<1>(p, t, cb, {&p.y});
            u32x4 r[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD && i < NV; ++i) {
                r[i] = ahead.template load<ST, TALL>(0, i, t, res);
                ahead.c.next();
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const u32x4 now = r[i % AHEAD];
                if (i + AHEAD < NV) {
                    r[i % AHEAD] = ahead.template load<ST, TALL>(0, i + AHEAD, t, res);
                    ahead.c.next();
                }
                if (TALL || i < t.count) put(v[i], &now, c.at[0]);
                c.next();
            }
        } else {
            GnCursor<1> c = gn_again<1>(p, t, cb, {&p.y});
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (TALL || i < t.count) put(v[i], nullptr, c.at[0]);
                c.next();
            }
        }
        if constexpr (TALL) {
            int from = t.first + NV * t.step, left = max(t.count - NV, 0);
            asm volatile("" : "+v"(from), "+v"(left)::"memory");  // not worked out ahead: the registers are full until here
            const int there = min(left, GN_KEPT_FWD);
            GnCursor<1> cy(from, t.step, p.W, cb, {&p.y});
            GnCursor<1> cx(from + there * t.step, t.step, p.W, cb, {&p.x});
            if (residual) {
                GnCursor<1> cr(from, t.step, p.W, cb, {&p.r});
                int i = 0;
                gn_pipelined<2, 1>(
                    there,
                    [&](u32x4* r) {
                        r[0] = gn_load<ST>(res, cr.at[0]);
                        cr.next();
                    },
                    [&](const u32x4* r) {
                        put(kept[i][threadIdx.x], r, cy.at[0]);
                        cy.next();
                        ++i;
                    });
                gn_pipelined<2, 2>(
                    left - there,
                    [&](u32x4* r) {
                        r[0] = gn_load<ST>(x, cx.at[0]);
                        r[1] = gn_load<ST>(res, cr.at[0]);
                        cx.next();
                        cr.next();
                    },
                    [&](const u32x4* r) {
                        put(r[0], r + 1, cy.at[0]);
                        cy.next();
                    });
            } else {
                for (int i = 0; i < there; ++i) {
                    put(kept[i][threadIdx.x], nullptr, cy.at[0]);
                    cy.next();
                }
                gn_pipelined<2, 1>(
                    left - there,
                    [&](u32x4* r) {
                        r[0] = gn_load<ST>(x, cx.at[0]);
                        cx.next();
                    },
                    [&](const u32x4* r) {
                        put(r[0], nullptr, cy.at[0]);
                        cy.next();
                    });
            }
        }
    });
}

// The backward pass the same way: x and dy in registers, the slab's sums per channel (they are also the image's share of dgamma
// and dbeta), the group's two terms, dx.  Four channels at a time, so that the constants of a channel stay few.  In this form
//   t = (x - mean) * (gamma r) + beta,   dx = d * (gamma r) - (x - mean) * (r r B) - r A.
//
// 64 x 13 x 13 x 1024 bf16: 66 MB in 21 us (one round of 512 workgroups that load, add up and store together), and 4 us for dgamma and
// dbeta under a profiler; the call takes 22 us.
//
// TALL: slabs that do not fit.  A thread's first NV pairs of vectors are in registers, the next GN_KEPT in LDS, and what is left
// is read again for dx; those beyond NV are summed first, eight channels at a time, as long as the registers are free.  The call on
// 64 x 52 x 52 x 256 bf16, 12 of a thread's 21 or 22 pairs held, takes 68 us, in chunks 83.  Eight pairs in registers spill a dozen
// values in bf16 (leaky) and are still no slower than seven or six (68.4, 68.1, 68.7 us; 64 x 38 x 38 x 512: 79.9, 81.2, 80.4).
constexpr int GN_KEPT = 4;
template <typename E, int ACT, int NV, bool TALL = false>
__global__ void __launch_bounds__(1024) gn_whole_bwd_kernel(const GnParams p) {
    constexpr int V = GnVec<E>::N, HALVES = V / 4;
    __shared__ u32x4 kept[TALL ? GN_KEPT : 1][2][TALL ? 1024 : 1];
    enum { MEAN, R, GAMMA, BETA, C0, C1, KINDS };
    __shared__ float part[2][GN_WAVES][GN_SLAB];
    __shared__ float chan[2][GN_SLAB];
    __shared__ __attribute__((aligned(16))) float of[KINDS][GN_SLAB];  // by channel
    const GnSeat t = gn_seat<E>(p);
    const int n = t.n, S = p.VS * V, c0 = t.slab * S, top = gn_top(p.PL), width = min(S, p.C - c0);
    const int groups = width / p.Cg;
    const int cb = (t.on ? t.c : 0) * (int)sizeof(E);
    {   // these loads come back first
        const int mine = min((int)threadIdx.x, width - 1), g = (c0 + mine) / p.Cg;
        const float mean = p.stats[n * p.groups + g], r = p.stats[(p.N + n) * p.groups + g];
        const float gamma = p.gamma[c0 + mine], beta = p.beta[c0 + mine];
        if ((int)threadIdx.x < width) {
            of[MEAN][mine] = mean;
            of[R][mine] = r;
            of[GAMMA][mine] = gamma;
            of[BETA][mine] = beta;
        }
    }
    const char* xp = p.x.p + n * p.x.img;
    const char* dp = p.dy.p + n * p.dy.img;
    float sd8[V], sx8[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sd8[e] = sx8[e] = 0.f;
    const int more = TALL ? max(t.count - NV, 0) : 0;
    if constexpr (TALL) {
        __syncthreads();
        const GnConst<V> k(&of[0][0] + t.cs, GN_SLAB);
        const float near = gn_near<V>(k.beta);
        GnCursor<2> c(t.first + NV * t.step, t.step, p.W, cb, {&p.x, &p.dy});
        int i = 0;
        gn_pipelined<2, 2>(
            more,
            [&](u32x4* r) {
                r[0] = gn_load(xp, c.at[0]);
                r[1] = gn_load(dp, c.at[1]);
                c.next();
            },
            [&](const u32x4* r) {
                if (i < GN_KEPT) {
                    kept[i][0][threadIdx.x] = r[0];
                    kept[i][1][threadIdx.x] = r[1];
                }
                ++i;
                float xm[V], a[V];
                gn_grads<E, ACT>(r[0], r[1], k, near, &of[0][0], t.cs, GN_SLAB, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sd8[e] += a[e];
                    sx8[e] = fmaf(a[e], xm[e], sx8[e]);
                }
            });
    }
    u32x4 x[NV], d[NV];
    gn_with_stream(p.stream, [&](auto st) {
        GnWalk<2> walk(p, t, cb, {&p.x, &p.dy});
#pragma unroll
        for (int i = 0; i < NV; ++i) {  // in turn: the first pairs are used while the last ones are on their way
            x[i] = walk.template load<decltype(st)::value, false>(0, i, t, xp);
            d[i] = walk.template load<decltype(st)::value, false>(1, i, t, dp);
            walk.c.next();
        }
    });
    gn_blank<NV>(d, t);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        if (h) {
            gn_forget<NV>(x);
            gn_forget<NV>(d);
        }
        const int cs = t.cs + 4 * h;
        const GnConst<4> k(&of[0][0] + cs, GN_SLAB);
        const float near = gn_near<4>(k.beta);
        float sd[4], sx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sd[e] = sd8[4 * h + e];
            sx[e] = sx8[4 * h + e];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < t.most) {  // where the thread has no pixel dy is zero
                float xm[4], a[4];
                gn_grads_of<E, ACT, 4>(x[i], d[i], h, k, near, &of[0][0], cs, GN_SLAB, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sd[e] += a[e];
                    sx[e] = fmaf(a[e], xm[e], sx[e]);
                }
            }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = gn_over_pixels(sd[e], p, t.pl, top), b = gn_over_pixels(sx[e], p, t.pl, top);
            if (t.pl == 0 && t.on) {
                part[0][t.wave][t.cs + 4 * h + e] = a;
                part[1][t.wave][t.cs + 4 * h + e] = b;
            }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * width; j += blockDim.x) {
        const int which = j >= width, c = j - which * width;
        float a = 0.f;
        for (int w = 0; w < t.waves; ++w) a += part[which][w][c];
        if (which) a *= of[R][c];
        chan[which][c] = a;
        p.sums[((long long)n * 2 + which) * p.C + c0 + c] = a;
    }
    __syncthreads();
    const int sub = threadIdx.x & 15;
    for (int h0 = 0; h0 < groups; h0 += blockDim.x >> 4) {
        const int g = h0 + (threadIdx.x >> 4);
        double A = 0.0, B = 0.0;
        if (g < groups)
            for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) {
                const double gamma = of[GAMMA][i];
                A += gamma * (double)chan[0][i];
                B += gamma * (double)chan[1][i];
            }
        for (int o = 8; o; o >>= 1) {
            A += __shfl_xor(A, o);
            B += __shfl_xor(B, o);
        }
        if (g < groups)
            for (int i = g * p.Cg + sub; i < (g + 1) * p.Cg; i += 16) {
                const double r = of[R][i];
                of[C0][i] = (float)(-r * (A * p.inv_count));
                of[C1][i] = (float)(-r * r * (B * p.inv_count));
            }
    }
    __syncthreads();
    if (!t.count) return;
    char* y = p.y.p + n * p.y.img;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        gn_forget<NV>(x);
        gn_forget<NV>(d);
        const int cs = t.cs + 4 * h;
        const GnConst<4> k(&of[0][0] + cs, GN_SLAB);
        const float near = gn_near<4>(k.beta);
        float k0[4], k1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k0[e] = of[C0][cs + e];
            k1[e] = of[C1][cs + e];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < t.most) {
                float xm[4], a[4];
                gn_grads_of<E, ACT, 4>(x[i], d[i], h, k, near, &of[0][0], cs, GN_SLAB, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = fmaf(a[e], k.scale[e], fmaf(xm[e], k1[e], k0[e]));
                gn_put_four<E>(x[i], h, a);
            }
    }
    gn_with_stream(p.stream, [&](auto st) {
        GnCursor<1> c = gn_again<1>(p, t, cb, {&p.y});
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i < t.count) gn_store<decltype(st)::value>(y, c.at[0], x[i]);
            c.next();
        }
    });
    if constexpr (TALL) {
        const GnConst<V> k(&of[0][0] + t.cs, GN_SLAB);
        const float near = gn_near<V>(k.beta);
        float k0[V], k1[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            k0[e] = of[C0][t.cs + e];
            k1[e] = of[C1][t.cs + e];
        }
        gn_with_stream(p.stream, [&](auto st) {
            constexpr int ST = decltype(st)::value;
            const int there = min(more, GN_KEPT);
            GnCursor<1> cy(t.first + NV * t.step, t.step, p.W, cb, {&p.y});
            GnCursor<2> c(t.first + (NV + there) * t.step, t.step, p.W, cb, {&p.x, &p.dy});
            auto put = [&](const u32x4* r) {
                float xm[V], a[V];
                gn_grads<E, ACT>(r[0], r[1], k, near, &of[0][0], t.cs, GN_SLAB, p.slope, xm, a);
#pragma unroll
                for (int e = 0; e < V; ++e) a[e] = fmaf(a[e], k.scale[e], fmaf(xm[e], k1[e], k0[e]));
                gn_store<ST>(y, cy.at[0], GnVec<E>::pack(a));
                cy.next();
            };
            for (int i = 0; i < there; ++i) {
                const u32x4 r[2] = {kept[i][0][threadIdx.x], kept[i][1][threadIdx.x]};
                put(r);
            }
            gn_pipelined<2, 2>(
                more - there,
                [&](u32x4* r) {
                    r[0] = gn_load<ST>(xp, c.at[0]);
                    r[1] = gn_load<ST>(dp, c.at[1]);
                    c.next();
                },
                put);
        });
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

// An output over an input: all of it in place, or none of it.
static int gn_check_overlap(const yolo_view* out, const yolo_view* in, int N, int C, int es, const char* op, const char* what) {
    const bool same = out->ch_total == in->ch_total && out->halo == in->halo;
    if (out->ptr == in->ptr && same &&
        (out->ch_offset == in->ch_offset || out->ch_offset + C <= in->ch_offset || in->ch_offset + C <= out->ch_offset))
        return YOLO_OK;
    auto bytes = [&](const yolo_view* v) { return (uintptr_t)N * (v->H + 2 * v->halo) * (v->W + 2 * v->halo) * v->ch_total * es; };
    const uintptr_t a = (uintptr_t)out->ptr, b = (uintptr_t)in->ptr;
    YOLO_REQUIRE(a + bytes(out) <= b || b + bytes(in) <= a, "%s: the output lies over part of %s", op, what);
    return YOLO_OK;
}

// What a call reads and writes beside its views has memory of its own.  (An output view over an input one: gn_check_overlap.)
struct GnRange {
    const char* what;
    const void* p;
    size_t bytes;
    bool written, view;
};
static GnRange gn_range(const char* what, const yolo_view* v, int N, int es, bool written) {
    return GnRange{what, v->ptr, (size_t)N * (v->H + 2 * v->halo) * (v->W + 2 * v->halo) * v->ch_total * es, written, true};
}
template <int K>
static int gn_check_memory(const GnRange (&r)[K], const char* op) {
    for (int i = 0; i < K; ++i)
        for (int j = 0; j < i; ++j) {
            const uintptr_t a = (uintptr_t)r[i].p, b = (uintptr_t)r[j].p;
            if (!a || !b || (r[i].view && r[j].view) || !(r[i].written || r[j].written)) continue;
            YOLO_REQUIRE(a + r[i].bytes <= b || b + r[j].bytes <= a, "%s: %s and %s share memory", op, r[j].what, r[i].what);
        }
    return YOLO_OK;
}

static GnTensor gn_tensor(const yolo_view* v, int es) {
    const ViewGeom g = geom_of(*v);
    return GnTensor{(char*)v->ptr + (long long)g.origin * es, g.img_stride * es, g.row_stride * es, g.pix_stride * es};
}

static int gn_check_shape(int N, int C, int groups, int act, float slope, int dtype, const char* op) {
    YOLO_REQUIRE(dtype == YOLO_F32 || dtype == YOLO_BF16, "%s: dtype %d", op, dtype);
    YOLO_REQUIRE(N > 0 && N <= 65534, "%s: batch %d (1 to 65534)", op, N);
    YOLO_REQUIRE(C > 0 && C % 8 == 0 && C <= 65536, "%s: %d channels (a multiple of 8, at most 65536)", op, C);
    YOLO_REQUIRE(groups > 0 && C % groups == 0, "%s: %d groups do not divide %d channels", op, groups, C);
    YOLO_REQUIRE(2ll * N * groups < (1ll << 31), "%s: %d images of %d groups (below 2^30 together)", op, N, groups);
    YOLO_REQUIRE(act == YOLO_ACT_LEAKY || act == YOLO_ACT_SILU, "%s: activation %d", op, act);
    YOLO_REQUIRE(act != YOLO_ACT_LEAKY || (slope >= 0.f && slope <= 1.f), "%s: leaky slope %g outside [0, 1]", op, (double)slope);
    return YOLO_OK;
}

static int gn_unit(const GnParams& p, int V) {  // vectors of the smallest slab: whole groups, whole vectors
    int unit = p.Cg;
    while (unit % V) unit += p.Cg;
    return unit / V;
}

// The split of an image over workgroups: pixel chunks so that about 2048 workgroups (8 per CU) are there, but no more than 256
// chunks for that (what joins them reads them all), no fewer than 4 pixels to a thread, and no more than 128 (its fp32 sums).
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
    if (chunk > 128ll * p.PL) chunk = 128ll * p.PL;
    p.chunk = (int)chunk;
    p.chunks = (int)((p.HW + chunk - 1) / chunk);
}

// The split for chunked passes without the joining launch: slabs of whole groups, about 128 B of a pixel, with so few chunks that a
// workgroup of the second pass reads no more than 64 KB of sums.  For up to 32 MB of x, and workgroups that are short or many
// (measured, bf16, us, with the joining launch and without):
//   8 x 104 x 104 x 128 forward with a residual 30.6 and 26.9;  16 images (44 MB) 43.2 and 44.6;  8 x 80 x 80 x 128 backward 23.9 and 21.2
//   1 x 104 x 104 x 64 (64 workgroups of 5 pixels a thread) forward 14.4 and 13.8;  1 x 208 x 208 x 64 (of 21 pixels) 18.5 and 22.6
static bool gn_split_joined(GnParams& p, int es, bool backward) {
    const int V = 16 / es, vecs = p.C / V, uv = gn_unit(p, V);
    if (uv > 32) return false;
    const int VS = uv > 8 ? uv : (vecs < 8 ? vecs : 8) / uv * uv, PL = GN_THREADS / VS, slabs = (vecs + VS - 1) / VS;
    const int most = 65536 / (2 * VS * V * (backward ? 4 : 8));
    long long want = 2048 / ((long long)p.N * slabs);
    if (want < 1) want = 1;
    if (want > most) want = most;
    long long chunk = (p.HW + want - 1) / want;
    if (chunk < 4ll * PL) chunk = 4ll * PL;
    if (chunk > 128ll * PL) return false;
    const long long chunks = (p.HW + chunk - 1) / chunk;
    if ((long long)p.N * p.HW * p.C * es > (32ll << 20) || (chunk > 16ll * PL && p.N * slabs * chunks < 512)) return false;
    p.VS = VS;
    p.PL = PL;
    p.chunk = (int)chunk;
    p.chunks = (int)chunks;
    p.stream = p.stream && (VS % 8 == 0 || VS == vecs);
    return !backward || (long long)p.N * p.chunks <= 512;  // rows that dgamma and dbeta are summed over
}

// Whether (and how) workgroups can hold the slabs of an image.  The slab's width, in bytes of a pixel, decides how whole the cache
// lines are that a workgroup reads, its height in registers what fits; measured (bf16, 32 groups, time of one call in us):
//   256 B where that leaves 512 workgroups       64 x 13 x 13 x 1024 backward 21.4, with 128 B 22.5
//   128 B otherwise                              64 x 52 x 52 x 256 forward 40, with 64 B 50, in chunks 56
//   narrower (to 32 B) for 256 workgroups        16 x 52 x 52 x 256 forward 16.1 with 32 B, 17.4 with 64 B, in chunks 22.3
//   64 B so that it fits, no less                64 x 104 x 104 x 128 forward 107 with 32 B, in chunks 96
// Forward a thread takes up to 11 vectors before the workgroup gets more waves (64 x 26 x 26 x 512: 18.1 us with 8 waves of 11, 23.3
// with 16 of 6); backward it has two tensors' vectors, and spills above 8.  Taller slabs are then held in part, at 128 B a pixel,
// where the CUs, one slab each, are busy:
//   backward, half of the CUs and more, to 32    64 x 52 x 52 x 256 68.0, in chunks 83;  32 images 44 and 52;  16 images 37 and 32
//                                                64 x 40 x 40 x 256 41, with 64 B whole 64
//   all of them, up to 64 vectors                64 x 76 x 76 x 256 backward 150, in chunks 161;  64 x 76 x 76 x 128 (128 slabs) 91 and 87
//                                                64 x 76 x 76 x 256 forward 83, in chunks 103;  64 x 88 x 88 x 256 126 and 133
//   several slabs each, the last round not empty 96 x 52 x 52 x 256 backward (384 slabs) 110, in chunks 117;  80 images (320) 104 and 99
struct GnWhole {
    int VS, waves, NV;
    bool tall;
};
static bool gn_whole_plan(const GnParams& p, int es, bool backward, GnWhole* out) {
    const int V = 16 / es, vecs = p.C / V;
    const int uv = gn_unit(p, V), most = GN_SLAB / V < vecs ? GN_SLAB / V : vecs;
    if (uv > most) return false;
    const int nv_many = backward ? 6 : 11, nv_most = backward ? 8 : 22;
    auto fit = [&](int vs) { return vs < uv ? uv : (vs < most ? vs : most) / uv * uv; };  // whole units, about vs vectors
    auto blocks = [&](int vs) { return (long long)p.N * ((vecs + vs - 1) / vs); };
    auto nv = [&](int vs, int waves) { return (p.HW + waves * (64 / vs) - 1) / (waves * (64 / vs)); };
    out->tall = false;
    int VS = fit(16);
    if (blocks(VS) < 512 || nv(VS, GN_WAVES) > nv_most) VS = fit(8);
    const long long there = blocks(VS), rounds = (there + 255) / 256;  // a tall slab takes a CU of its own
    const int tall = nv(VS, GN_WAVES);
    const bool busy = there <= 256 ? there >= (backward && tall <= 32 ? 128 : 256) : there * 10 >= rounds * 256 * 7;
    if (tall > nv_most && tall <= 64 && (VS % 8 == 0 || VS == vecs) && busy) {
        *out = GnWhole{VS, GN_WAVES, tall, true};
        return true;
    }
    if (tall > nv_most) VS = fit(4);
    if (nv(VS, GN_WAVES) > nv_most) return false;
    if (blocks(VS) < 256 && VS > 4) VS = fit(4);
    if (blocks(VS) < 256 && VS > 2) VS = fit(2);
    int waves = 4;
    while (waves < GN_WAVES && nv(VS, waves) > nv_many) waves *= 2;
    out->VS = VS;
    out->waves = waves;
    out->NV = nv(VS, waves);
    return true;
}

// Where both are possible, the chunked passes without the joining launch have every CU at work on few images, and whole slabs x in
// registers.  Measured (us, whole and chunked; forward: replays of a graph over three sets of buffers):
//   forward, with a residual: 48 KB and more to each of less than 256 workgroups: 1 x 52 x 52 x 256 11.4 and 9.6, 8 images 17.9 and
//             16.2, 16 (256 workgroups) 19.3 and 25.1;  4 x 60 x 60 x 128 14.7 and 11.8;  1 x 40 x 40 x 256 (56 KB) 9.1 and 9.6, 1 x 26 x
//             26 x 512 (28 KB) 7.5 and 9.6
//   without one: 80 KB, less than 32: 1 x 52 x 52 x 256 10.1 and 9.5, 8 images 13.8 and 15.7;  1 x 40 x 40 x 256 8.2 and 9.5
//             112 KB, less than 128: 8 x 64 x 64 x 64 (64) 15.3 and 11.8;  16 x 60 x 60 x 128 (128) 16.9 and 17.6
//   backward  bf16, less than 512 slabs of 128 B: 1 x 40 x 40 x 256 20.8 and 11.0, 24 x 13 x 13 x 1024 (384) 17.8 and 17.0, 32 (512) 18.9
//             and 19.9;  16 MB and less: 16 x 26 x 26 x 512 20.0 and 18.6, 32 (22 MB) 26.6 and 29.9
//             f32, less than 128: 4 x 26 x 26 x 512 (64) 13.4 and 13.2, 8 x 13 x 13 x 1024 (256) 11.8 and 13.1
static bool gn_whole_first(const GnParams& p, int es, bool backward, const GnWhole& w) {
    const int vecs = p.C * es / 16;
    if (w.tall) return true;
    if (!backward) {
        const int kb = w.waves * w.NV, few = p.r.p ? (kb >= 48 ? 256 : 0) : (kb >= 112 ? 128 : kb >= 80 ? 32 : 0);
        return (long long)p.N * ((vecs + w.VS - 1) / w.VS) >= few;
    }
    return (long long)p.N * ((vecs + 7) / 8) >= (es == 2 ? 512 : 128) || (long long)p.N * p.HW * p.C * es > (16ll << 20);
}

// A call that moves more than this leaves little of use in the 256 MB cache in front of HBM; its loads and stores go past the
// caches, and what the first pass over x has left there stays for the second.  Measured (bf16, us): 64 x 208 x 208 x 64 forward
// 229 -> 192, backward 347 -> 306; 64 x 52 x 52 x 256 forward 53 -> 40; 64 x 13 x 13 x 1024 backward (66 MB) 23.0 -> 21.8; the
// one that lost, 16 x 104 x 104 x 128 forward (88 MB): 36.1 -> 36.5.  A network's training step takes the same time with either.
// Only where a workgroup's stores are whole cache lines: narrower slabs share them, and lose a factor of two and more.
constexpr long long GN_STREAM_BYTES = 64ll << 20;
static int gn_stream_rule(const GnParams& p, int es, int tensors) {
    return (long long)tensors * p.N * p.HW * p.C * es >= GN_STREAM_BYTES;
}

// The channels of a vector that always lie in one group: the largest power of two that divides both.
static int gn_fold(int Cg, int V) {
    int f = 1;
    while (f < V && Cg % (2 * f) == 0) f *= 2;
    return f;
}

// The form of a call, with the split that goes with it: p holds the chunked one of three launches.  *held: vectors a thread of the
// whole form has in registers, the instance to launch.
enum GnForm { GN_FORM_WHOLE, GN_FORM_TALL, GN_FORM_JOINED, GN_FORM_CHUNKED };
static GnForm gn_form(GnParams& p, int es, bool backward, GnWhole* w, int* held) {
    p.stream = gn_stream_rule(p, es, backward || p.r.p ? 3 : 2);
    GnParams q = p;
    const bool joined = gn_split_joined(q, es, backward);
    if (!gn_whole_plan(p, es, backward, w) || (joined && !gn_whole_first(p, es, backward, *w))) {
        if (joined) p = q;
        return joined ? GN_FORM_JOINED : GN_FORM_CHUNKED;
    }
    p.VS = w->VS;
    p.PL = 64 / w->VS;
    p.fold = gn_fold(p.Cg, 16 / es);
    p.slabs = (p.C * es / 16 + w->VS - 1) / w->VS;
    p.stream = p.stream && w->VS % 8 == 0;  // whole cache lines only
    static const int fwd[] = {1, 2, 4, 6, 8, 11, 16, 22}, bwd[] = {1, 2, 4, 6, 8};
    const int* k = backward ? bwd : fwd;
    while (!w->tall && *k < w->NV) ++k;  // gn_whole_plan keeps to the last one
    *held = !w->tall ? *k : backward ? 8 : 12;
    return w->tall ? GN_FORM_TALL : GN_FORM_WHOLE;
}

static dim3 gn_join_grid(const GnParams& p) {
    const int per = p.Cg < 64 ? 64 / p.Cg : 1;
    return dim3((p.groups + per - 1) / per, p.N);
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

// KERNEL for the call's type and activation; what follows are its other template arguments
#define GN_LAUNCH(grid, block, KERNEL, ...)                                                                  \
    do {                                                                                                     \
        if (dtype == YOLO_BF16 && act == YOLO_ACT_LEAKY)                                                     \
            hipLaunchKernelGGL((KERNEL<unsigned short, GN_LEAKY, ##__VA_ARGS__>), grid, block, 0, st, p);    \
        else if (dtype == YOLO_BF16)                                                                         \
            hipLaunchKernelGGL((KERNEL<unsigned short, GN_SILU, ##__VA_ARGS__>), grid, block, 0, st, p);     \
        else if (act == YOLO_ACT_LEAKY)                                                                      \
            hipLaunchKernelGGL((KERNEL<float, GN_LEAKY, ##__VA_ARGS__>), grid, block, 0, st, p);             \
        else                                                                                                 \
            hipLaunchKernelGGL((KERNEL<float, GN_SILU, ##__VA_ARGS__>), grid, block, 0, st, p);              \
    } while (0)

#define GN_WHOLE_CASE(KERNEL, K)                          \
    if (held == K)                                        \
        GN_LAUNCH(grid, dim3(w.waves * 64), KERNEL, K);   \
    else

extern "C" size_t yolo_gn_workspace_bytes(int N, int H, int W, int C, int groups, int dtype) {
    if (N <= 0 || H <= 0 || W <= 0 || C <= 0 || C % 8 || groups <= 0 || C % groups || (long long)H * W >= (1ll << 31)) return 0;
    GnParams p{};
    yolo_view v{nullptr, H, W, 0, C, 0};
    const int es = (int)elem_size(dtype);
    gn_shape(p, &v, N, C, groups, es);
    // forward: the double sums, then the pivots; backward: the float sums, then the images' sums and the groups' terms
    auto sums = [&](const GnParams& q, size_t size) { return (size_t)N * q.chunks * 2 * C * size; };
    size_t most = sums(p, sizeof(float)) + ((size_t)N * 2 * C + (size_t)2 * N * groups) * sizeof(float);
    auto more = [&](size_t bytes) { most = bytes > most ? bytes : most; };
    const size_t pivots = (size_t)N * C * sizeof(float);
    more(sums(p, sizeof(double)) + pivots);
    GnParams q = p;
    if (gn_split_joined(q, es, false)) more(sums(q, sizeof(double)) + pivots);
    if (gn_split_joined(q, es, true)) more(sums(q, sizeof(float)));
    return most;
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
    if (int e = gn_check_overlap(y, x, N, C, es, "gn_act_fwd", "x")) return e;
    if (residual)
        if (int e = gn_check_overlap(y, residual, N, C, es, "gn_act_fwd", "residual")) return e;
    YOLO_REQUIRE((uintptr_t)workspace % 16 == 0, "gn_act_fwd: workspace is not 16-byte aligned");
    const size_t need = yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype), vec = (size_t)C * 4;
    if (ws_bytes < need) return fail(YOLO_E_WORKSPACE, "gn_act_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
    const GnRange memory[] = {gn_range("x", x, N, es, false), gn_range("y", y, N, es, true),
                              residual ? gn_range("residual", residual, N, es, false) : GnRange{},
                              {"gamma", gamma, vec, false, false}, {"beta", beta, vec, false, false},
                              {"stats", stats, (size_t)N * groups * 8, true, false}, {"workspace", workspace, need, true, false}};
    if (int e = gn_check_memory(memory, "gn_act_fwd")) return e;
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
    GnWhole w;
    int held;
    const GnForm form = gn_form(p, es, false, &w, &held);
    if (form == GN_FORM_WHOLE || form == GN_FORM_TALL) {
        const dim3 grid((unsigned)(p.slabs * N));
        if (w.tall && residual)
            GN_LAUNCH(grid, dim3(1024), gn_whole_kernel, 12, GN_TALL_RESIDUAL);
        else if (w.tall)
            GN_LAUNCH(grid, dim3(1024), gn_whole_kernel, 12, GN_TALL);
        else
        GN_WHOLE_CASE(gn_whole_kernel, 1)
        GN_WHOLE_CASE(gn_whole_kernel, 2)
        GN_WHOLE_CASE(gn_whole_kernel, 4)
        GN_WHOLE_CASE(gn_whole_kernel, 6)
        GN_WHOLE_CASE(gn_whole_kernel, 8)
        GN_WHOLE_CASE(gn_whole_kernel, 11)
        GN_WHOLE_CASE(gn_whole_kernel, 16)
        GN_WHOLE_CASE(gn_whole_kernel, 22) { return fail(YOLO_E_ARG, "gn_act_fwd: no kernel for %d vectors", w.NV); }
        YOLO_CHECK_HIP(hipGetLastError());
        return YOLO_OK;
    }
    p.pivots = (float*)((double*)workspace + (size_t)N * p.chunks * 2 * C);
    const dim3 grid = gn_grid(p, es);
    if (dtype == YOLO_BF16)
        hipLaunchKernelGGL((gn_sums_kernel<unsigned short>), grid, dim3(GN_THREADS), 0, st, p);
    else
        hipLaunchKernelGGL((gn_sums_kernel<float>), grid, dim3(GN_THREADS), 0, st, p);
    if (form == GN_FORM_JOINED) {
        GN_LAUNCH(grid, dim3(GN_THREADS), gn_apply_kernel, true);
    } else {
        hipLaunchKernelGGL(gn_join_kernel<false>, gn_join_grid(p), dim3(GN_JOIN * 64), 0, st, p);
        GN_LAUNCH(grid, dim3(GN_THREADS), gn_apply_kernel);
    }
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
    if (int e = gn_check_overlap(dx, x, N, C, es, "gn_act_bwd", "x")) return e;
    if (int e = gn_check_overlap(dx, dy, N, C, es, "gn_act_bwd", "dy")) return e;
    YOLO_REQUIRE(dgamma != dbeta && dgamma != gamma && dgamma != beta && dbeta != gamma && dbeta != beta,
                 "gn_act_bwd: dgamma and dbeta need memory of their own");
    YOLO_REQUIRE((uintptr_t)workspace % 16 == 0, "gn_act_bwd: workspace is not 16-byte aligned");
    const size_t need = yolo_gn_workspace_bytes(N, x->H, x->W, C, groups, dtype), vec = (size_t)C * 4;
    if (ws_bytes < need) return fail(YOLO_E_WORKSPACE, "gn_act_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
    const GnRange memory[] = {gn_range("x", x, N, es, false), gn_range("dy", dy, N, es, false), gn_range("dx", dx, N, es, true),
                              {"gamma", gamma, vec, false, false}, {"beta", beta, vec, false, false},
                              {"stats", stats, (size_t)N * groups * 8, false, false}, {"dgamma", dgamma, vec, true, false},
                              {"dbeta", dbeta, vec, true, false}, {"workspace", workspace, need, true, false}};
    if (int e = gn_check_memory(memory, "gn_act_bwd")) return e;
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
    GnWhole w;
    int held;
    const GnForm form = gn_form(p, es, true, &w, &held);
    if (form == GN_FORM_WHOLE || form == GN_FORM_TALL) {
        const dim3 grid((unsigned)(p.slabs * N));
        if (w.tall)
            GN_LAUNCH(grid, dim3(1024), gn_whole_bwd_kernel, 8, true);
        else
        GN_WHOLE_CASE(gn_whole_bwd_kernel, 1)
        GN_WHOLE_CASE(gn_whole_bwd_kernel, 2)
        GN_WHOLE_CASE(gn_whole_bwd_kernel, 4)
        GN_WHOLE_CASE(gn_whole_bwd_kernel, 6)
        GN_WHOLE_CASE(gn_whole_bwd_kernel, 8) { return fail(YOLO_E_ARG, "gn_act_bwd: no kernel for %d vectors", w.NV); }
        hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((2 * C + 31) / 32), dim3(GN_THREADS), 0, st, p);
        YOLO_CHECK_HIP(hipGetLastError());
        return YOLO_OK;
    }
    const bool joined = form == GN_FORM_JOINED;
    dim3 grid = gn_grid(p, es);
    GN_LAUNCH(grid, dim3(GN_THREADS), gn_bwd_sums_kernel);
    if (!joined) hipLaunchKernelGGL(gn_join_kernel<true>, gn_join_grid(p), dim3(GN_JOIN * 64), 0, st, p);
    ++grid.z;  // dgamma and dbeta
    if (joined)
        GN_LAUNCH(grid, dim3(GN_THREADS), gn_bwd_apply_kernel, true);
    else
        GN_LAUNCH(grid, dim3(GN_THREADS), gn_bwd_apply_kernel);
    YOLO_CHECK_HIP(hipGetLastError());
    return YOLO_OK;
}

extern "C" int yolo_gn_kernel_name(int N, int H, int W, int C, int groups, int dtype, int residual, int backward, char* out, int out_len) {
    YOLO_REQUIRE(out && out_len > 0, "gn_kernel_name: bad argument");
    if (int e = gn_check_shape(N, C, groups, YOLO_ACT_LEAKY, 0.f, dtype, "gn_kernel_name")) return e;
    const int es = (int)elem_size(dtype);
    YOLO_REQUIRE(H > 0 && W > 0 && (long long)H * W < (1ll << 31) / C / es, "gn_kernel_name: %d x %d x %d", H, W, C);
    GnParams p{};
    const yolo_view v{nullptr, H, W, 0, C, 0};
    gn_shape(p, &v, N, C, groups, es);
    p.r.p = residual && !backward ? out : nullptr;  // whether there is one is all that counts
    GnWhole w;
    int held = 0;
    const GnForm form = gn_form(p, es, backward != 0, &w, &held);
    static const char* const forms[] = {"whole", "tall", "joined", "chunked"};
    char many[16] = "";
    if (held) snprintf(many, sizeof many, ",%d", held);
    snprintf(out, (size_t)out_len, "gn_%s%skernel<%s%s,%s%s>", held ? "whole_" : "", backward ? "bwd_" : "", dtype == YOLO_BF16 ? "bf16" : "float",
             many, forms[form], p.stream ? ",stream" : "");
    return YOLO_OK;
}
