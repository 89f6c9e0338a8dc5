// Group norm with SiLU or without, and its gradients:
//
//   xh = (x - mean) rstd over a group of channels and all pixels of an image,
//   z = gamma_c xh + beta_c,  y = z or z sigmoid(z)
//   dz = dy or dy (s + z s (1 - s)), s = sigmoid(z)
//   dbeta_c = sum dz, dgamma_c = sum dz xh over images and pixels
//   dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh)) over the group
//
// Bytes bound it: x is read and y written once at least, and the statistics of
// a group stand between the two. Three forms:
//
//   one launch   a workgroup holds whole groups of one image in registers
//                (up to 128 KB)
//   pieces       a launch sums pieces of the image, another joins the pieces'
//                statistics and writes y; the pieces are the same, so the
//                second read of x finds much of it in the caches
//   plain        a workgroup per group, element by element: channel counts
//                that the others' thread layouts do not take
//
// One launch against pieces, us (without the gap between two launches): 1280
// channels @8^2 5.0 | 10.5, 2 x 640 @16^2 9.3 | 12.7, 512 @32^2 7.2 | 10.2, 2 x
// 320 @32^2 13.4 | 12.5, where 16 workgroups hold it all; NCHW 2 x 320 @32^2
// 7.0 | 8.5. Chains of dependent steps bound it at these sizes: the loads, two
// sums over the workgroup, the stores.
// Pieces, us and what the launches move (float16): 128 channels @512^2 statistics
// 16, join 4, y 23 (67 MB read, 134 MB read and written: 4.2 and 5.8 TB/s, the
// second with help of the memory-side cache); 8 x 320 @64^2 statistics 11.5, y
// 12, sums 14.3, join 4, dx 14.5 (21 MB a tensor: 1.8, 3.5, 2.9 and 4.3 TB/s),
// whose workgroups live for one or two trips to memory.
//
// The variance is summed about a mean: a workgroup's own, from registers, or a
// thread's running one, and pieces are joined by count, mean and squared
// deviations. No sum of squares loses digits to a large mean or to an outlier.
// All sums are float32.
//
// Channels-last: a thread owns V neighbouring channels (up to 16 bytes) and
// walks pixels, so its gamma and beta stay in registers. NCHW: lanes share a
// channel's row and walk its 16-byte pieces.
#include <algorithm>
#include <type_traits>

#include "nova_internal.h"

namespace nova {

namespace {

constexpr int kThreads = 256;
constexpr int kWide = 1024;  // threads where a row of channels needs them, or a slab does
constexpr int kStream = 4;   // vectors that a thread has in flight per tensor: x alone ...
constexpr int kPair = 2;     // ... or x and dy
constexpr int kJoin = 64;    // pieces that every workgroup of the next launch joins for itself

// x / d for x and d below 2^16: the compiler's own division by a runtime value
// takes some 40 dependent instructions, and a small image's workgroup lives for
// a few thousand cycles.
struct Div {
    unsigned inv;
    int d;
    __device__ __forceinline__ int quot(int x) const {
        return inv == 0 ? x : (int)__umulhi((unsigned)x, inv);
    }
};
Div div_by(int d) {
    return Div{d <= 1 ? 0u : (unsigned)((((uint64_t)1 << 32) + d - 1) / d), std::max(d, 1)};
}

struct GnArgs {
    const void *x, *dy, *gamma, *beta;
    void *y, *dgamma, *dbeta;
    float *mean, *rstd;
    float* part;  // forward: [B][G (NCHW: C)][pieces] of (count, mean, squares); backward:
                  // [B][pieces][2][C] sums of dz and dz xh, then [B][2][C] of all pieces
    float* sums;  // backward: [B][G][2], means of gamma dz and gamma dz xh
    int B, C, G, n, params, nhwc, silu;
    int P;
    int pieces, per;  // pieces of an image; pixels (vectors of a row) in each
    int rows;         // channels-last: pixels that a workgroup takes at a time
    int lanes_c;      // channels-last: lanes of a wave across channels (the others: pixels)
    int tiles;        // channels-last: waves across channels
    int threads;      // channels-last: of the workgroup
    int lanes;        // NCHW: lanes of a row
    int grid;         // workgroups of the launch that writes dx, without params_done's
    int sets;         // channels-last, one launch: workgroups of an image
    int share;        // channels-last: lanes that add up one group's values
    int span;         // channels-last: groups that the workgroup adds up at a time
    int cols;         // channels-last: vectors per pixel that a workgroup owns
    Div width;        // channels of a group
    Div across;       // channels-last: a group's values in a row of threads
    float eps;
    // channels-last: waves above one another
    __host__ __device__ int bands() const { return rows * lanes_c / 64; }
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <typename T, int V>
struct Pair {
    Pack<T, V> x, d;
};

__device__ __forceinline__ float param(const void* p, int type, int c, float none) {
    if (p == nullptr) return none;
    if (type == kF16) return (float)static_cast<const _Float16*>(p)[c];
    if (type == kBF16) return (float)static_cast<const __bf16*>(p)[c];
    return static_cast<const float*>(p)[c];
}

// N parameters, all in flight at once: one branch on the type around the loads
// (a branch and a wait for each made up most of a small image's time).
template <int N>
__device__ __forceinline__ void params(const void* p, int type, const int (&at)[N], float none,
                                       float (&out)[N]) {
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = none;
    } else if (type == kF32) {
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = static_cast<const float*>(p)[at[i]];
    } else {
        uint16_t raw[N];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = static_cast<const uint16_t*>(p)[at[i]];
        if (type == kF16) {
#pragma unroll
            for (int i = 0; i < N; i++) out[i] = (float)__builtin_bit_cast(_Float16, raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) out[i] = (float)__builtin_bit_cast(__bf16, raw[i]);
        }
    }
}

// gamma and beta of V neighbouring channels, and the groups they are in.
template <int V>
struct Channels {
    float w[V], b[V];
    int group[V];
    __device__ __forceinline__ Channels(const GnArgs& a, int c) {
        int at[V], g = a.width.quot(c), end = (g + 1) * a.n;
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (c + j >= end) {
                g++;
                end += a.n;
            }
            group[j] = g;
            at[j] = c + j;
        }
        params(a.gamma, a.params, at, 1.0f, w);
        params(a.beta, a.params, at, 0.0f, b);
    }
};

__device__ __forceinline__ void store_param(void* p, int type, int c, float v) {
    if (type == kF16) static_cast<_Float16*>(p)[c] = (_Float16)v;
    else if (type == kBF16) static_cast<__bf16*>(p)[c] = (__bf16)v;
    else static_cast<float*>(p)[c] = v;
}

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

__device__ __forceinline__ float activate(float z, int silu) {
    return silu ? z * sigmoid(z) : z;
}

// dz for a value's xh and dy.
__device__ __forceinline__ float grad_z(float xh, float w, float bb, float d, int silu) {
    if (!silu) return d;
    const float z = __builtin_fmaf(xh, w, bb), s = sigmoid(z);
    return d * __builtin_fmaf(z * s, 1.0f - s, s);
}

__device__ __forceinline__ float rstd_of(float sq, float n, float eps) {
    return 1.0f / __builtin_sqrtf(sq / n + eps);
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                             0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Sum over `lanes` neighbouring lanes (1 to 64, a power of two, the same in the
// whole wave), in every one of them: within 16 by lane permutations of the adds
// themselves, then by the rows' totals from scalar registers. No trip through
// LDS.
__device__ __forceinline__ float sum_lanes(float v, int lanes) {
    if (lanes >= 2) v = add_dpp<0xB1>(v);   // lane ^ 1
    if (lanes >= 4) v = add_dpp<0x4E>(v);   // lane ^ 2
    if (lanes >= 8) v = add_dpp<0x141>(v);  // mirrored in 8
    if (lanes >= 16) v = add_dpp<0x140>(v); // mirrored in 16
    if (lanes >= 32) {
        const float lo = lane_value(v, 0) + lane_value(v, 16);
        const float hi = lane_value(v, 32) + lane_value(v, 48);
        v = lanes == 64 ? lo + hi : (threadIdx.x & 32) ? hi : lo;
    }
    return v;
}

// Sum over the lanes of a wave whose numbers agree modulo w (a power of two, the
// same in the whole wave), in every one of them.
__device__ __forceinline__ float sum_strided(float v, int w) {
    // swapping halves between two copies of v leaves its lower half in both
    // halves of one, its upper half in both of the other
    if (w < 64) {
        const int u = __builtin_bit_cast(int, v);
        const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (int)x[0]) + __builtin_bit_cast(float, (int)x[1]);
    }
    if (w < 32) {
        const int u = __builtin_bit_cast(int, v);
        const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (int)x[0]) + __builtin_bit_cast(float, (int)x[1]);
    }
    if (w < 16) v = add_dpp<0x128>(v);  // rotated by 8 in 16 lanes
    if (w < 8) v = add_dpp<0x124>(v);
    if (w < 4) v = add_dpp<0x122>(v);
    if (w < 2) v = add_dpp<0x121>(v);
    return v;
}

// Sum over the workgroup, the same in every thread.
template <int TH>
__device__ __forceinline__ float sum_all(float v, float* lds) {
    v = sum_lanes(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < TH / 64; w++) s += lds[w];
    return s;
}

// Walks [at, end) in steps, R items at a time, the next R on their way while
// use(items, at, valid) takes the current ones (the first `valid` of them).
template <int R, typename Item, typename Load, typename Use>
__device__ __forceinline__ void stream(int at, int end, int step, Load load, Use use) {
    Item now[R], next[R];
#pragma unroll
    for (int i = 0; i < R; i++)
        if (at + i * step < end) now[i] = load(at + i * step);
    while (at < end) {
        const int then = at + R * step;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (then + i * step < end) next[i] = load(then + i * step);
        int valid = 1;
#pragma unroll
        for (int i = 1; i < R; i++) valid += at + i * step < end;
        use(now, at, valid);
#pragma unroll
        for (int i = 0; i < R; i++) now[i] = next[i];
        at = then;
    }
}

// ---- sums of the backward, both layouts --------------------------------------

// From the pieces' sums, a workgroup per group and image: the image's sums per
// channel, and the means that dx needs. Every sum in a fixed order.
__global__ __launch_bounds__(kThreads) void sums_join_kernel(GnArgs a) {
    __shared__ float lds[2][kThreads], red[2][kThreads / 64];
    const int tid = threadIdx.x;
    const int b = blockIdx.x / a.G, g = blockIdx.x % a.G;
    float* all = a.part + 2 * (int64_t)a.B * a.pieces * a.C + 2 * (int64_t)b * a.C;
    const int wide = min(a.n, kThreads), parts = kThreads / wide;
    const int col = tid % wide, part = tid / wide;
    float s1 = 0.0f, s2 = 0.0f;
    for (int c0 = 0; c0 < a.n; c0 += wide) {
        const bool ok = part < parts && c0 + col < a.n;
        const int c = g * a.n + c0 + col;
        float s = 0.0f, t = 0.0f;
        if (ok) {
            const float* q = a.part + 2 * (int64_t)b * a.pieces * a.C + c;
#pragma unroll 4
            for (int i = part; i < a.pieces; i += parts) {
                s += q[2 * (int64_t)i * a.C];
                t += q[(2 * (int64_t)i + 1) * a.C];
            }
        }
        __syncthreads();
        lds[0][tid] = s;
        lds[1][tid] = t;
        __syncthreads();
        if (ok && part == 0) {
#pragma unroll 4
            for (int k = 1; k < parts; k++) {
                s += lds[0][tid + wide * k];
                t += lds[1][tid + wide * k];
            }
            all[c] = s;
            all[a.C + c] = t;
            const float w = param(a.gamma, a.params, c, 1.0f);
            s1 = __builtin_fmaf(w, s, s1);
            s2 = __builtin_fmaf(w, t, s2);
        }
    }
    s1 = sum_all<kThreads>(s1, red[0]);
    s2 = sum_all<kThreads>(s2, red[1]);
    if (tid == 0) {
        const float of = 1.0f / ((float)a.n * (float)a.P);
        a.sums[2 * (int64_t)blockIdx.x] = s1 * of;
        a.sums[2 * (int64_t)blockIdx.x + 1] = s2 * of;
    }
}

// The gradients of gamma and beta from the images' sums, in the last
// workgroups of the launch that writes dx (64 channels each): true where the
// workgroup is one of them.
constexpr int kParamChannels = 64;
__device__ __forceinline__ bool params_done(const GnArgs& a, int first) {
    if ((int)blockIdx.x < first) return false;
    __shared__ float lds[2][kWide];
    const int tid = threadIdx.x, c = ((int)blockIdx.x - first) * kParamChannels + (tid & 63);
    float s = 0.0f, t = 0.0f;
    if (c < a.C) {
        const float* q = a.part + 2 * (int64_t)a.B * a.pieces * a.C + c;
#pragma unroll 4
        for (int b = tid >> 6; b < a.B; b += a.threads / 64) {
            s += q[2 * (int64_t)b * a.C];
            t += q[(2 * (int64_t)b + 1) * a.C];
        }
    }
    lds[0][tid] = s;
    lds[1][tid] = t;
    __syncthreads();
    if (tid < 64 && c < a.C) {
        for (int k = 1; k < a.threads / 64; k++) {
            s += lds[0][tid + 64 * k];
            t += lds[1][tid + 64 * k];
        }
        store_param(a.dbeta, a.params, c, s);
        store_param(a.dgamma, a.params, c, t);
    }
    return true;
}

// ---- channels-last ---------------------------------------------------------

// A thread's place: vector `col` of the workgroup's channels, pixel `row` of
// those that it takes at a time. A wave spans lanes_c vectors and 64 / lanes_c
// pixels, so the pixels' sums stay in registers; `tiles` waves span the
// channels, `band` counts the waves above one another.
struct Spot {
    int col, row, band;
    bool first;  // of its wave's pixels
    __device__ __forceinline__ explicit Spot(const GnArgs& a) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int lane = threadIdx.x & 63, high = 64 / a.lanes_c;
        band = wave / a.tiles;
        col = (wave - band * a.tiles) * a.lanes_c + (lane & (a.lanes_c - 1));
        const int up = lane / a.lanes_c;
        row = band * high + up;
        first = up == 0;
    }
};

// Adds every thread's V values of its channels over the pixels and the channels
// of each group; out[g] (LDS) holds fin(total, g) for each of the workgroup's
// `groups` groups. red: bands * cols * V floats. Inactive threads bring zeros. A
// group's values are shared by up to 64 neighbouring lanes, so no thread walks
// a long column of them alone. MANY: groups may outnumber the threads.
template <int V, bool MANY, typename F>
__device__ __forceinline__ void group_totals(float (&v)[V], const Spot& at, const GnArgs& a,
                                             int groups, float* red, float* out, F fin) {
    const bool single = a.across.d < a.n || V == 1;  // a thread's channels are of one group
    const int width = single ? a.cols : a.cols * V;
    __syncthreads();
    if (single) {
#pragma unroll
        for (int j = 1; j < V; j++) v[0] += v[j];
        v[0] = sum_strided(v[0], a.lanes_c);
        if (at.first && at.col < a.cols) red[at.band * width + at.col] = v[0];
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = sum_strided(v[j], a.lanes_c);
        if (at.first && at.col < a.cols)
#pragma unroll
            for (int j = 0; j < V; j++) red[at.band * width + at.col * V + j] = v[j];
    }
    __syncthreads();
    const int lanes = a.share, per = a.across.d, bands = a.bands();
    const int l = threadIdx.x & (lanes - 1);
    for (int g = threadIdx.x / lanes; g < groups; g += a.span) {
        float s = 0.0f;
        int r = a.across.quot(l), c = l - r * per;
        const int dr = a.across.quot(lanes), dc = lanes - dr * per;
        for (int i = l; i < per * bands; i += lanes) {
            s += red[r * width + g * per + c];
            r += dr;
            c += dc;
            if (c >= per) {
                c -= per;
                r++;
            }
        }
        s = sum_lanes(s, lanes);
        if (l == 0) out[g] = fin(s, g);
        if (!MANY) break;
    }
    __syncthreads();
}

// One launch: the workgroup's channels hold whole groups, its pixels the image.
template <typename T, int V, int R, int TH>
__global__ __launch_bounds__(TH) void norm_nhwc_one_kernel(GnArgs a) {
    __shared__ float red[TH * V], total[TH];
    typedef Pack<T, V> P;
    const Spot spot(a);
    const int row = spot.row;
    const bool active = spot.col < a.cols;
    const int b = blockIdx.x / a.sets, set = blockIdx.x - b * a.sets;
    const int c0 = set * a.cols * V, c = c0 + (active ? spot.col : 0) * V;
    const T* x = static_cast<const T*>(a.x) + (int64_t)b * a.P * a.C + c;
    const int g0 = a.width.quot(c0), groups = a.width.quot(a.cols * V);

    P v[R];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int p = row + i * a.rows;
        if (active && p < a.P) {
            v[i] = *reinterpret_cast<const P*>(x + (int64_t)p * a.C);
            mine++;
        }
    }
    Channels<V> ch(a, c);
    float s[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        s[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (i < mine) s[j] += (float)v[i].v[j];
    }
    const float count = (float)a.n * (float)a.P, part = 1.0f / count;
    const int64_t at = (int64_t)b * a.G + g0;
    group_totals<V, false>(s, spot, a, groups, red, total, [&](float t, int g) {
        const float m = t * part;
        a.mean[at + g] = m;
        return m;
    });
    float mean[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        mean[j] = total[ch.group[j] - g0];
        s[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (i < mine) {
                const float d = (float)v[i].v[j] - mean[j];
                s[j] = __builtin_fmaf(d, d, s[j]);
            }
    }
    group_totals<V, false>(s, spot, a, groups, red, total, [&](float t, int g) {
        const float r = rstd_of(t, count, a.eps);
        a.rstd[at + g] = r;
        return r;
    });
    if (!active) return;
#pragma unroll
    for (int j = 0; j < V; j++) ch.w[j] *= total[ch.group[j] - g0];
    T* y = static_cast<T*>(a.y) + (int64_t)b * a.P * a.C + c;
#pragma unroll
    for (int i = 0; i < R; i++)
        if (i < mine) {
            P o;
#pragma unroll
            for (int j = 0; j < V; j++)
                o.v[j] = (T)activate(
                    __builtin_fmaf((float)v[i].v[j] - mean[j], ch.w[j], ch.b[j]), a.silu);
            *reinterpret_cast<P*>(y + (int64_t)(row + i * a.rows) * a.C) = o;
        }
}

// A thread's channels and pixels (first, a.rows on, up to end) in a piece.
template <int V>
struct Place {
    Spot spot;
    int b, piece, p0, p1, c;
    bool active;
    __device__ __forceinline__ explicit Place(const GnArgs& a) : spot(a) {
        active = spot.col < a.cols;
        b = blockIdx.x / a.pieces;
        piece = blockIdx.x - b * a.pieces;
        p0 = piece * a.per;
        p1 = min(a.P, p0 + a.per);
        c = active ? spot.col * V : 0;
    }
    __device__ __forceinline__ int64_t base(const GnArgs& a) const {
        return (int64_t)b * a.P * a.C + c;
    }
    __device__ __forceinline__ int first() const { return p0 + spot.row; }
    __device__ __forceinline__ int end() const { return active ? p1 : 0; }
};

// Statistics of a piece's groups. A thread keeps a running mean and squared
// deviations of each of its channels, kStream pixels at a time.
template <typename T, int V, bool MANY>
__global__ __launch_bounds__(kWide) void stats_nhwc_kernel(GnArgs a) {
    extern __shared__ float lds[];  // bands * C, then G
    float *red = lds, *total = lds + a.bands() * a.C;
    typedef Pack<T, V> P;
    const Place<V> at(a);
    const T* x = static_cast<const T*>(a.x) + at.base(a);
    float m[V], q[V];
    float n = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) m[j] = q[j] = 0.0f;
    stream<kStream, P>(
        at.first(), at.end(), a.rows,
        [&](int p) { return *reinterpret_cast<const P*>(x + (int64_t)p * a.C); },
        [&](const P(&v)[kStream], int, int valid) {
            const float k = (float)valid, f = k / (n + k), of = 1.0f / k, both = n * f;
            auto take = [&](auto count) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float s = (float)v[0].v[j];
#pragma unroll
                    for (int i = 1; i < kStream; i++)
                        if (i < count) s += (float)v[i].v[j];
                    const float mine = s * of;
                    float sq = 0.0f;
#pragma unroll
                    for (int i = 0; i < kStream; i++)
                        if (i < count) {
                            const float d = (float)v[i].v[j] - mine;
                            sq = __builtin_fmaf(d, d, sq);
                        }
                    const float d = mine - m[j];
                    m[j] = __builtin_fmaf(d, f, m[j]);
                    q[j] += __builtin_fmaf(d * d, both, sq);
                }
            };
            if (valid == kStream) take(std::integral_constant<int, kStream>());
            else take(valid);
            n += k;
        });
    float s[V];
#pragma unroll
    for (int j = 0; j < V; j++) s[j] = m[j] * n;
    const float count = (float)a.n * (float)(at.p1 - at.p0), part = 1.0f / count;
    float* to = a.part + 3 * ((int64_t)at.b * a.G * a.pieces + at.piece);
    group_totals<V, MANY>(s, at.spot, a, a.G, red, total, [&](float t, int g) {
        const float mean = t * part;
        to[3 * (int64_t)g * a.pieces] = count;
        to[3 * (int64_t)g * a.pieces + 1] = mean;
        return mean;
    });
    int g = a.width.quot(at.c), end = (g + 1) * a.n;
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (at.c + j >= end) {
            g++;
            end += a.n;
        }
        const float d = m[j] - total[g];
        s[j] = __builtin_fmaf(d * d, n, q[j]);
    }
    group_totals<V, MANY>(s, at.spot, a, a.G, red, total, [&](float t, int g) {
        to[3 * (int64_t)g * a.pieces + 2] = t;
        return t;
    });
}

// Joins the statistics of a group's pieces, each (count, mean, squares) one
// after the other: `lanes` neighbours take every lanes-th piece, all get
// (mean, rstd).
__device__ __forceinline__ void join(const float* q, int pieces, int lane, int lanes, float eps,
                                     float* mean, float* rstd) {
    float n = 0.0f, s = 0.0f;
#pragma unroll 8
    for (int i = lane; i < pieces; i += lanes) {
        n += q[3 * i];
        s = __builtin_fmaf(q[3 * i], q[3 * i + 1], s);
    }
    n = sum_lanes(n, lanes);
    const float m = sum_lanes(s, lanes) / n;
    s = 0.0f;
#pragma unroll 8
    for (int i = lane; i < pieces; i += lanes) {
        const float d = q[3 * i + 1] - m;
        s += __builtin_fmaf(q[3 * i] * d, d, q[3 * i + 2]);
    }
    *mean = m;
    *rstd = rstd_of(sum_lanes(s, lanes), n, eps);
}

// mean and rstd of every group, where its pieces are too many for every
// workgroup of the next launch to join them again. each: pieces of a group.
__global__ __launch_bounds__(64) void norm_join_kernel(GnArgs a, int each) {
    const int at = blockIdx.x, lane = threadIdx.x;
    float mean, rstd;
    join(a.part + 3 * (int64_t)at * each, each, lane, 64, a.eps, &mean, &rstd);
    if (lane == 0) {
        a.mean[at] = mean;
        a.rstd[at] = rstd;
    }
}

// y of a piece. JOIN: the statistics come from the pieces'; otherwise from mean
// and rstd.
template <typename T, int V, bool JOIN>
__global__ __launch_bounds__(kWide) void apply_nhwc_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    __shared__ float sm[JOIN ? kWide : 1], sr[JOIN ? kWide : 1];
    const Place<V> at(a);
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + at.base(a);
    T* y = static_cast<T*>(a.y) + at.base(a);
    Channels<V> ch(a, at.c);
    float mean[V], rstd[V];
    if (JOIN) {
        // 8 lanes a group
        for (int g = tid / 8; g < a.G; g += a.threads / 8) {
            float m, r;
            join(a.part + 3 * ((int64_t)at.b * a.G + g) * a.pieces, a.pieces, tid & 7, 8, a.eps,
                 &m, &r);
            if ((tid & 7) == 0) {
                sm[g] = m;
                sr[g] = r;
                if (at.piece == 0) {
                    a.mean[(int64_t)at.b * a.G + g] = m;
                    a.rstd[(int64_t)at.b * a.G + g] = r;
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        mean[j] = JOIN ? sm[ch.group[j]] : a.mean[(int64_t)at.b * a.G + ch.group[j]];
        rstd[j] = JOIN ? sr[ch.group[j]] : a.rstd[(int64_t)at.b * a.G + ch.group[j]];
    }
#pragma unroll
    for (int j = 0; j < V; j++) ch.w[j] *= rstd[j];
    stream<kStream, P>(
        at.first(), at.end(), a.rows,
        [&](int p) { return *reinterpret_cast<const P*>(x + (int64_t)p * a.C); },
        [&](const P(&v)[kStream], int p, int valid) {
#pragma unroll
            for (int i = 0; i < kStream; i++)
                if (i < valid) {
                    P o;
#pragma unroll
                    for (int j = 0; j < V; j++)
                        o.v[j] = (T)activate(
                            __builtin_fmaf((float)v[i].v[j] - mean[j], ch.w[j], ch.b[j]), a.silu);
                    *reinterpret_cast<P*>(y + (int64_t)(p + i * a.rows) * a.C) = o;
                }
        });
}

// Sums of dz and dz xh per channel over a piece of pixels.
template <typename T, int V>
__global__ __launch_bounds__(kWide) void sums_nhwc_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    typedef Pair<T, V> Two;
    extern __shared__ float red[];  // 2 * bands * C
    const Place<V> at(a);
    const T* x = static_cast<const T*>(a.x) + at.base(a);
    const T* dy = static_cast<const T*>(a.dy) + at.base(a);
    const Channels<V> ch(a, at.c);
    float mean[V], rstd[V], s[V], t[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        mean[j] = a.mean[(int64_t)at.b * a.G + ch.group[j]];
        rstd[j] = a.rstd[(int64_t)at.b * a.G + ch.group[j]];
        s[j] = t[j] = 0.0f;
    }
    stream<kPair, Two>(
        at.first(), at.end(), a.rows,
        [&](int p) {
            return Two{*reinterpret_cast<const P*>(x + (int64_t)p * a.C),
                       *reinterpret_cast<const P*>(dy + (int64_t)p * a.C)};
        },
        [&](const Two(&v)[kPair], int, int valid) {
#pragma unroll
            for (int i = 0; i < kPair; i++)
                if (i < valid)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xh = ((float)v[i].x.v[j] - mean[j]) * rstd[j];
                        const float z =
                            grad_z(xh, ch.w[j], ch.b[j], (float)v[i].d.v[j], a.silu);
                        s[j] += z;
                        t[j] = __builtin_fmaf(z, xh, t[j]);
                    }
        });
#pragma unroll
    for (int j = 0; j < V; j++) {
        s[j] = sum_strided(s[j], a.lanes_c);
        t[j] = sum_strided(t[j], a.lanes_c);
    }
    const int bands = a.bands();
    if (at.spot.first && at.active)
#pragma unroll
        for (int j = 0; j < V; j++) {
            red[at.spot.band * a.C + at.c + j] = s[j];
            red[(bands + at.spot.band) * a.C + at.c + j] = t[j];
        }
    __syncthreads();
    float* to = a.part + 2 * ((int64_t)at.b * a.pieces + at.piece) * a.C;
    for (int i = threadIdx.x; i < 2 * a.C; i += a.threads) {
        const int which = i >= a.C, c = i - which * a.C;
        float u = 0.0f;
        for (int r = 0; r < bands; r++) u += red[(which * bands + r) * a.C + c];
        to[i] = u;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kWide) void dx_nhwc_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    typedef Pair<T, V> Two;
    if (params_done(a, a.grid)) return;
    const Place<V> at(a);
    const T* x = static_cast<const T*>(a.x) + at.base(a);
    const T* dy = static_cast<const T*>(a.dy) + at.base(a);
    T* dx = static_cast<T*>(a.y) + at.base(a);
    const Channels<V> ch(a, at.c);
    float mean[V], rstd[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int64_t g = (int64_t)at.b * a.G + ch.group[j];
        mean[j] = a.mean[g];
        rstd[j] = a.rstd[g];
        s1[j] = a.sums[2 * g];
        s2[j] = a.sums[2 * g + 1];
    }
    stream<kPair, Two>(
        at.first(), at.end(), a.rows,
        [&](int p) {
            return Two{*reinterpret_cast<const P*>(x + (int64_t)p * a.C),
                       *reinterpret_cast<const P*>(dy + (int64_t)p * a.C)};
        },
        [&](const Two(&v)[kPair], int p, int valid) {
#pragma unroll
            for (int i = 0; i < kPair; i++)
                if (i < valid) {
                    P o;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xh = ((float)v[i].x.v[j] - mean[j]) * rstd[j];
                        const float z =
                            grad_z(xh, ch.w[j], ch.b[j], (float)v[i].d.v[j], a.silu);
                        o.v[j] =
                            (T)(rstd[j] * (__builtin_fmaf(ch.w[j], z, -s1[j]) - xh * s2[j]));
                    }
                    *reinterpret_cast<P*>(dx + (int64_t)(p + i * a.rows) * a.C) = o;
                }
        });
}

// ---- NCHW ------------------------------------------------------------------

// A row of P elements from element `start` of the tensor, cut where V elements
// align: vector i holds the row's elements i * V - shift on. A row's first and
// last vector may hold elements of its neighbours: loads bring them along
// (inside() tells them apart), stores leave them out.
template <typename T, int V>
struct Row {
    int64_t start;
    int shift, P;
    __device__ __forceinline__ Row(int64_t s, int p) : start(s), shift((int)(s % V)), P(p) {}
    __device__ __forceinline__ int vectors() const { return (P + shift + V - 1) / V; }
    __device__ __forceinline__ int first(int i) const { return i * V - shift; }
    __device__ __forceinline__ bool whole(int i) const {
        return first(i) >= 0 && first(i) + V <= P;
    }
    __device__ __forceinline__ int count(int i) const {
        return min(first(i) + V, P) - max(first(i), 0);
    }
    __device__ __forceinline__ bool inside(int i, int j) const {
        const int e = first(i) + j;
        return e >= 0 && e < P;
    }
    // all: elements of the tensor, whose last vector may reach past its end
    __device__ __forceinline__ Pack<T, V> load(const T* x, int i, int64_t all) const {
        Pack<T, V> v;
        const int64_t e = start + first(i);
        if (e + V <= all) {
            v = *reinterpret_cast<const Pack<T, V>*>(x + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) v.v[j] = e + j < all ? x[e + j] : (T)0.0f;
        }
        return v;
    }
    __device__ __forceinline__ void store(T* y, int i, const Pack<T, V>& v) const {
        const int e = first(i);
        if (whole(i)) {
            *reinterpret_cast<Pack<T, V>*>(y + start + e) = v;
            return;
        }
#pragma unroll
        for (int j = 0; j < V; j++)
            if (e + j >= 0 && e + j < P) y[start + e + j] = v.v[j];
    }
    // f(value) over the row's elements of vector i
    template <typename F>
    __device__ __forceinline__ void each(int i, const Pack<T, V>& v, F f) const {
        if (whole(i)) {
#pragma unroll
            for (int j = 0; j < V; j++) f((float)v.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (inside(i, j)) f((float)v.v[j]);
        }
    }
};

// One launch: a workgroup per group, its rows in registers. A thread's slots
// walk the vectors of a row `lanes` apart, then the row `rows` further down.
template <typename T, int V, int R, int TH>
__global__ __launch_bounds__(TH) void norm_nchw_one_kernel(GnArgs a) {
    __shared__ float lds[TH / 64];
    typedef Pack<T, V> P;
    const int tid = threadIdx.x, lane = tid & (a.lanes - 1), sub = tid / a.lanes;
    const int g = blockIdx.x % a.G, b = blockIdx.x / a.G;
    const int rows = TH / a.lanes;
    const int64_t base = ((int64_t)b * a.G + g) * a.n * a.P;
    const int64_t all = (int64_t)a.B * a.C * a.P - base;
    const T* x = static_cast<const T*>(a.x) + base;
    T* y = static_cast<T*>(a.y) + base;
    const float count = (float)a.n * (float)a.P;
    const int lead = (int)(base % V);  // elements in front of the group in its first vector
    P v[R];
    int off[R], lo[R], hi[R], c[R];  // the slot's vector in the group; its elements of the row
    int r = sub, at = lane;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int start = r * a.P, shift = (start + lead) % V;
        const int e = at * V - shift;  // first element, in the row
        off[i] = start + e;
        lo[i] = max(-e, 0);
        hi[i] = r < a.n ? min(a.P - e, V) : 0;
        c[i] = g * a.n + min(r, a.n - 1);
        if (lo[i] < hi[i]) {
            if (off[i] + V <= all) {
                v[i] = *reinterpret_cast<const P*>(x + off[i]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    v[i].v[j] = j < hi[i] ? x[off[i] + j] : (T)0.0f;
            }
        }
        at += a.lanes;
        if (at >= a.per) {  // vectors of a row at most, rounded up to the lanes
            at = lane;
            r += rows;
        }
    }
    float w[R], bb[R];
    params(a.gamma, a.params, c, 1.0f, w);
    params(a.beta, a.params, c, 0.0f, bb);
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            if (hi[i] - lo[i] == V) {
#pragma unroll
                for (int j = 0; j < V; j++) f((float)v[i].v[j]);
            } else if (lo[i] < hi[i]) {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (j >= lo[i] && j < hi[i]) f((float)v[i].v[j]);
            }
        }
    };
    float s = 0.0f;
    each([&](float e) { s += e; });
    const float mean = sum_all<TH>(s, lds) / count;
    s = 0.0f;
    each([&](float e) { s = __builtin_fmaf(e - mean, e - mean, s); });
    const float rstd = rstd_of(sum_all<TH>(s, lds), count, a.eps);
    if (tid == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        if (lo[i] >= hi[i]) continue;
        P o;
        const float scale = w[i] * rstd;
#pragma unroll
        for (int j = 0; j < V; j++)
            o.v[j] = (T)activate(__builtin_fmaf((float)v[i].v[j] - mean, scale, bb[i]), a.silu);
        if (hi[i] - lo[i] == V) {
            *reinterpret_cast<P*>(y + off[i]) = o;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j >= lo[i] && j < hi[i]) y[off[i] + j] = o.v[j];
        }
    }
}

// The row, and the vectors [i0, i1) of it, that a thread's lanes share.
template <typename T, int V>
struct Span {
    int b, c, piece, lane, i0, i1;
    bool ok;
    __device__ __forceinline__ explicit Span(const GnArgs& a) {
        const int rows = kThreads / a.lanes;
        const int block = blockIdx.x / a.pieces;
        piece = blockIdx.x - block * a.pieces;
        lane = threadIdx.x & (a.lanes - 1);
        const int r = block * rows + threadIdx.x / a.lanes;
        ok = r < a.B * a.C;
        b = ok ? r / a.C : 0;
        c = ok ? r - b * a.C : 0;
        i0 = piece * a.per;
        i1 = ok ? min(row(a).vectors(), i0 + a.per) : 0;
    }
    __device__ __forceinline__ Row<T, V> row(const GnArgs& a) const {
        return Row<T, V>(((int64_t)b * a.C + c) * a.P, a.P);
    }
};

// Statistics of a piece of a row: part[b][c][piece].
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void stats_nchw_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    const Span<T, V> sp(a);
    const Row<T, V> row = sp.row(a);
    const int64_t all = (int64_t)a.B * a.C * a.P;
    const T* x = static_cast<const T*>(a.x);
    float n = 0.0f, m = 0.0f, q = 0.0f;
    stream<kStream, P>(
        sp.i0 + sp.lane, sp.i1, a.lanes, [&](int i) { return row.load(x, i, all); },
        [&](const P(&v)[kStream], int i0, int valid) {
            float k = 0.0f, s = 0.0f, sq = 0.0f;
#pragma unroll
            for (int i = 0; i < kStream; i++)
                if (i < valid) {
                    k += (float)row.count(i0 + i * a.lanes);
                    row.each(i0 + i * a.lanes, v[i], [&](float e) { s += e; });
                }
            const float mine = s / k, f = k / (n + k), d = mine - m;
#pragma unroll
            for (int i = 0; i < kStream; i++)
                if (i < valid)
                    row.each(i0 + i * a.lanes, v[i],
                             [&](float e) { sq = __builtin_fmaf(e - mine, e - mine, sq); });
            m = __builtin_fmaf(d, f, m);
            q += __builtin_fmaf(d * d, n * f, sq);
            n += k;
        });
    // the lanes': about their common mean
    const float count = sum_lanes(n, a.lanes);
    const float mean = count > 0.0f ? sum_lanes(m * n, a.lanes) / count : 0.0f;
    const float squares = sum_lanes(__builtin_fmaf((m - mean) * (m - mean), n, q), a.lanes);
    if (sp.ok && sp.lane == 0) {
        float* to = a.part + 3 * (((int64_t)sp.b * a.C + sp.c) * a.pieces + sp.piece);
        to[0] = count;
        to[1] = mean;
        to[2] = squares;
    }
}

template <typename T, int V, bool JOIN>
__global__ __launch_bounds__(kThreads) void apply_nchw_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    const Span<T, V> sp(a);
    const Row<T, V> row = sp.row(a);
    const int64_t all = (int64_t)a.B * a.C * a.P;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const int c[1] = {sp.c};
    float w[1], bb[1];
    params(a.gamma, a.params, c, 1.0f, w);
    params(a.beta, a.params, c, 0.0f, bb);
    const int g = sp.c / a.n;
    const int64_t at = (int64_t)sp.b * a.G + g;
    float mean, rstd;
    if (JOIN) {
        join(a.part + 3 * at * a.n * a.pieces, a.n * a.pieces, sp.lane, a.lanes, a.eps, &mean,
             &rstd);
        if (sp.ok && sp.lane == 0 && sp.piece == 0 && sp.c == g * a.n) {
            a.mean[at] = mean;
            a.rstd[at] = rstd;
        }
    } else {
        mean = a.mean[at];
        rstd = a.rstd[at];
    }
    const float scale = w[0] * rstd;
    stream<kStream, P>(
        sp.i0 + sp.lane, sp.i1, a.lanes, [&](int i) { return row.load(x, i, all); },
        [&](const P(&v)[kStream], int i0, int valid) {
#pragma unroll
            for (int i = 0; i < kStream; i++)
                if (i < valid) {
                    P o;
#pragma unroll
                    for (int j = 0; j < V; j++)
                        o.v[j] = (T)activate(
                            __builtin_fmaf((float)v[i].v[j] - mean, scale, bb[0]), a.silu);
                    row.store(y, i0 + i * a.lanes, o);
                }
        });
}

// What the backward kernels know of a row.
struct RowStats {
    float mean, rstd, w[1], b[1];
    int64_t group;
    __device__ __forceinline__ RowStats(const GnArgs& a, int image, int channel) {
        const int c[1] = {channel};
        group = (int64_t)image * a.G + channel / a.n;
        mean = a.mean[group];
        rstd = a.rstd[group];
        params(a.gamma, a.params, c, 1.0f, w);
        params(a.beta, a.params, c, 0.0f, b);
    }
};

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sums_nchw_kernel(GnArgs a) {
    typedef Pair<T, V> Two;
    const Span<T, V> sp(a);
    const Row<T, V> row = sp.row(a);
    const int64_t all = (int64_t)a.B * a.C * a.P;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const RowStats st(a, sp.b, sp.c);
    float s = 0.0f, t = 0.0f;
    stream<kPair, Two>(
        sp.i0 + sp.lane, sp.i1, a.lanes,
        [&](int i) {
            return Two{row.load(x, i, all), row.load(dy, i, all)};
        },
        [&](const Two(&v)[kPair], int i0, int valid) {
#pragma unroll
            for (int i = 0; i < kPair; i++)
                if (i < valid) {
                    const bool whole = row.whole(i0 + i * a.lanes);
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xh = ((float)v[i].x.v[j] - st.mean) * st.rstd;
                        const float z =
                            grad_z(xh, st.w[0], st.b[0], (float)v[i].d.v[j], a.silu);
                        if (whole || row.inside(i0 + i * a.lanes, j)) {
                            s += z;
                            t = __builtin_fmaf(z, xh, t);
                        }
                    }
                }
        });
    s = sum_lanes(s, a.lanes);
    t = sum_lanes(t, a.lanes);
    if (sp.ok && sp.lane == 0) {
        float* to = a.part + 2 * ((int64_t)sp.b * a.pieces + sp.piece) * a.C + sp.c;
        to[0] = s;
        to[a.C] = t;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void dx_nchw_kernel(GnArgs a) {
    typedef Pack<T, V> P;
    typedef Pair<T, V> Two;
    if (params_done(a, a.grid)) return;
    const Span<T, V> sp(a);
    const Row<T, V> row = sp.row(a);
    const int64_t all = (int64_t)a.B * a.C * a.P;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.y);
    const RowStats st(a, sp.b, sp.c);
    const float s1 = a.sums[2 * st.group], s2 = a.sums[2 * st.group + 1];
    stream<kPair, Two>(
        sp.i0 + sp.lane, sp.i1, a.lanes,
        [&](int i) {
            return Two{row.load(x, i, all), row.load(dy, i, all)};
        },
        [&](const Two(&v)[kPair], int i0, int valid) {
#pragma unroll
            for (int i = 0; i < kPair; i++)
                if (i < valid) {
                    P o;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xh = ((float)v[i].x.v[j] - st.mean) * st.rstd;
                        const float z =
                            grad_z(xh, st.w[0], st.b[0], (float)v[i].d.v[j], a.silu);
                        o.v[j] = (T)(st.rstd * (__builtin_fmaf(st.w[0], z, -s1) - xh * s2));
                    }
                    row.store(dx, i0 + i * a.lanes, o);
                }
        });
}

// ---- plain -----------------------------------------------------------------

// Element i of group g of image b, in the order of memory; *c: its channel.
__device__ __forceinline__ int64_t element(const GnArgs& a, int b, int g, int64_t i, int* c) {
    if (a.nhwc) {
        *c = g * a.n + (int)(i % a.n);
        return ((int64_t)b * a.P + i / a.n) * a.C + *c;
    }
    *c = g * a.n + (int)(i / a.P);
    return ((int64_t)b * a.C + g * a.n) * a.P + i;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_plain_kernel(GnArgs a) {
    __shared__ float lds[kThreads / 64];
    const int g = blockIdx.x % a.G, b = blockIdx.x / a.G;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const int64_t all = (int64_t)a.n * a.P;
    int c;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < all; i += kThreads) s += (float)x[element(a, b, g, i, &c)];
    const float mean = sum_all<kThreads>(s, lds) / (float)all;
    s = 0.0f;
    for (int64_t i = threadIdx.x; i < all; i += kThreads) {
        const float d = (float)x[element(a, b, g, i, &c)] - mean;
        s = __builtin_fmaf(d, d, s);
    }
    const float rstd = rstd_of(sum_all<kThreads>(s, lds), (float)all, a.eps);
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
    for (int64_t i = threadIdx.x; i < all; i += kThreads) {
        const int64_t e = element(a, b, g, i, &c);
        const float w = param(a.gamma, a.params, c, 1.0f) * rstd;
        const float bb = param(a.beta, a.params, c, 0.0f);
        y[e] = (T)activate(__builtin_fmaf((float)x[e] - mean, w, bb), a.silu);
    }
}

// Channel sums by a workgroup per channel and image (one piece).
template <typename T>
__global__ __launch_bounds__(kThreads) void sums_plain_kernel(GnArgs a) {
    __shared__ float lds[kThreads / 64];
    const int c = blockIdx.x % a.C, b = blockIdx.x / a.C;
    const int64_t g = (int64_t)b * a.G + c / a.n;
    const float mean = a.mean[g], rstd = a.rstd[g];
    const float w = param(a.gamma, a.params, c, 1.0f), bb = param(a.beta, a.params, c, 0.0f);
    const int64_t base = a.nhwc ? (int64_t)b * a.P * a.C + c : ((int64_t)b * a.C + c) * a.P;
    const int64_t step = a.nhwc ? a.C : 1;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* dy = static_cast<const T*>(a.dy) + base;
    float s = 0.0f, t = 0.0f;
    for (int p = threadIdx.x; p < a.P; p += kThreads) {
        const float xh = ((float)x[p * step] - mean) * rstd;
        const float z = grad_z(xh, w, bb, (float)dy[p * step], a.silu);
        s += z;
        t = __builtin_fmaf(z, xh, t);
    }
    s = sum_all<kThreads>(s, lds);
    t = sum_all<kThreads>(t, lds);
    if (threadIdx.x == 0) {
        float* q = a.part + 2 * (int64_t)b * a.C + c;
        q[0] = s;
        q[a.C] = t;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dx_plain_kernel(GnArgs a) {
    if (params_done(a, a.grid)) return;
    const int64_t all = (int64_t)a.B * a.C * a.P;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all;
         i += (int64_t)a.grid * kThreads) {
        const int64_t pixel = a.nhwc ? i / a.C : i / a.P;  // (b, p), or (b, c)
        const int c = (int)(a.nhwc ? i % a.C : pixel % a.C);
        const int64_t b = a.nhwc ? pixel / a.P : pixel / a.C, g = b * a.G + c / a.n;
        const float rstd = a.rstd[g], w = param(a.gamma, a.params, c, 1.0f);
        const float xh = ((float)static_cast<const T*>(a.x)[i] - a.mean[g]) * rstd;
        const float z = grad_z(xh, w, param(a.beta, a.params, c, 0.0f),
                               (float)static_cast<const T*>(a.dy)[i], a.silu);
        static_cast<T*>(a.y)[i] =
            (T)(rstd * (__builtin_fmaf(w, z, -a.sums[2 * g]) - xh * a.sums[2 * g + 1]));
    }
}

// ---- choice of the form ----------------------------------------------------

enum Form { kPlain, kOne, kPieces };

struct Plan {
    Form form;
    int V, R, TH;  // TH: threads of the workgroup
    bool join;     // a launch of its own joins the pieces
    int cols, lanes_c, tiles, rows, lanes, pieces, per, sets, share, across;
    int64_t grid;
};

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Vector length: elements of up to 16 bytes that every row starts on.
int vector_of(const GroupNorm& g, const void* const* ptrs, int n) {
    const int size = g.dtype == kF32 ? 4 : 2;
    int V = 16 / size;
    if (g.nhwc)
        while (g.C % V != 0) V /= 2;
    for (int i = 0; i < n; i++)
        while (V > 1 && reinterpret_cast<uintptr_t>(ptrs[i]) % (V * size) != 0) V /= 2;
    if (!g.nhwc && V * size != 16) V = 1;
    return V;
}

// Threads and registers of the one-launch form for a slab that takes `small`
// steps of kThreads threads, `large` of kWide; false where it does not fit.
bool one_fits(Plan* p, int64_t small, int64_t large, int most) {
    if (small <= 4) {
        p->TH = kThreads;
        p->R = small <= 2 ? 2 : 4;
        return true;
    }
    p->TH = kWide;
    p->R = large <= 4 ? 4 : 8;
    return large <= most;
}

// Channels-last: the threads' places for p->cols vectors and p->TH threads.
void place(Plan* p, int width, int groups) {
    p->rows = 64 / p->lanes_c * (p->TH / 64 / p->tiles);
    p->across = width % p->V == 0 ? width / p->V : width;
    p->share = 64;
    while (p->share > 1 && p->share * groups > p->TH) p->share /= 2;
}

Plan plan_of(const GroupNorm& g, const void* const* ptrs, int n, bool backward, int cus) {
    Plan p{};
    p.V = vector_of(g, ptrs, n);
    p.pieces = 1;
    const int width = g.C / g.G;
    if (g.nhwc) {
        const int nv = g.C / p.V;
        if (nv > kWide || g.G > kWide) {
            p.form = kPlain;
            return p;
        }
        // whole groups that are whole vectors
        int set = width;
        while (set % p.V != 0) set += width;
        if (!backward && g.C % set == 0 && set / p.V <= 64) {
            p.cols = set / p.V;
            p.lanes_c = 1;
            while (p.lanes_c < p.cols) p.lanes_c *= 2;
            p.tiles = 1;
            if (one_fits(&p, div_up(g.P, kThreads / p.lanes_c), div_up(g.P, kWide / p.lanes_c),
                         8)) {
                p.form = kOne;
                p.per = (int)g.P;
                p.sets = g.C / set;
                p.grid = (int64_t)g.B * p.sets;
                place(&p, width, set / width);
                return p;
            }
        }
        p.form = kPieces;
        p.cols = nv;
        // waves 8 vectors wide (128 bytes), wider where channels would take
        // more than a workgroup's 16
        p.lanes_c = 8;
        while (div_up(nv, p.lanes_c) > kWide / 64) p.lanes_c *= 2;
        p.tiles = (int)div_up(nv, p.lanes_c);
        auto waves = [&](int some) {
            int bands = std::max(1, some / p.tiles);
            // a thread for every group, where a workgroup holds that many
            while (64 * p.tiles * bands < g.G && 64 * p.tiles * (bands + 1) <= kWide) bands++;
            p.TH = 64 * p.tiles * bands;
            place(&p, width, g.G);
        };
        // Two workgroups of four waves or more for every CU: a wave's share of
        // the parameters and of the sums across lanes costs as much as some 60
        // of its elements (320 channels @64^2 batch 8, us, stats + apply + sums
        // + dx at 256, 512 and 1024 workgroups: 59, 52, 64).
        waves(4);
        const int deep = backward ? kPair : kStream;
        p.pieces = (int)std::min(div_up(2 * cus, g.B), div_up(g.P, p.rows * deep));
        // No more pieces than the next launch joins for itself, in workgroups
        // of ten waves, where that still gives half of the CUs work: one launch
        // less (@64^2 batch 2: 14.6 + a gap between launches -> 14.4).
        if (!backward && p.pieces > kJoin && g.B * kJoin >= cus / 2 &&
            g.P <= (int64_t)kJoin * p.rows * 16) {
            waves(10);
            p.pieces = (int)std::min<int64_t>(kJoin, div_up(g.P, p.rows));
        }
        p.per = (int)(div_up(div_up(g.P, p.pieces), p.rows) * p.rows);
        p.pieces = (int)div_up(g.P, p.per);
        p.join = p.pieces > kJoin;
        p.grid = (int64_t)g.B * p.pieces;
        return p;
    }
    const int64_t nv = div_up(g.P + p.V - 1, p.V);  // vectors of a row at most
    if (!backward && (int64_t)width * g.P < (1 << 30)) {
        int few = 8, many = 8;
        while (few < kThreads && few < nv) few *= 2;
        while (many < kWide && many < nv) many *= 2;
        if (one_fits(&p, div_up(nv, few) * div_up(width, kThreads / few),
                     div_up(nv, many) * div_up(width, kWide / many), 4)) {
            p.form = kOne;
            p.lanes = p.TH == kThreads ? few : many;
            p.per = (int)(div_up(nv, p.lanes) * p.lanes);
            p.grid = (int64_t)g.B * g.G;
            return p;
        }
    }
    p.form = kPieces;
    p.TH = kThreads;
    p.lanes = 8;
    while (p.lanes < 64 && p.lanes < nv) p.lanes *= 2;
    const int64_t blocks = div_up((int64_t)g.B * g.C, kThreads / p.lanes);
    const int64_t most = div_up(nv, (int64_t)p.lanes * (backward ? kPair : kStream));
    p.pieces = (int)std::max<int64_t>(1, std::min(div_up(8 * cus, blocks), most));
    p.per = (int)(div_up(div_up(nv, p.pieces), p.lanes) * p.lanes);
    p.pieces = (int)div_up(nv, p.per);
    p.join = (int64_t)width * p.pieces > 4 * kJoin;
    p.grid = blocks * p.pieces;
    return p;
}

// Workgroups of dx_plain_kernel, whose threads walk further than their own
// element where the tensor has more than that many.
int plain_grid(const GroupNorm& g) {
    return (int)std::min<int64_t>(div_up((int64_t)g.B * g.C * g.P, kThreads), 1 << 20);
}

int extra_of(const GroupNorm& g) { return (int)div_up(g.C, kParamChannels); }

GnArgs args_of(const GroupNorm& g, const Plan& p) {
    GnArgs a{};
    a.x = g.x;
    a.gamma = g.gamma;
    a.beta = g.beta;
    a.B = g.B;
    a.C = g.C;
    a.G = g.G;
    a.n = g.C / g.G;
    a.params = g.params;
    a.nhwc = g.nhwc;
    a.silu = g.silu;
    a.P = (int)g.P;
    a.eps = g.eps;
    a.pieces = p.pieces;
    a.per = p.per;
    a.rows = p.rows;
    a.lanes = p.lanes;
    a.grid = (int)p.grid;
    a.sets = p.sets;
    a.share = p.share;
    a.span = p.share > 0 ? p.TH / p.share : 0;
    a.cols = p.cols;
    a.lanes_c = p.lanes_c;
    a.tiles = p.tiles;
    a.threads = p.form == kPlain ? kThreads : p.TH;
    a.width = div_by(a.n);
    a.across = div_by(p.across);
    return a;
}

template <typename T, int V>
void one_v(const GroupNorm& g, const Plan& p, const GnArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)p.grid), block(p.TH);
    if (g.nhwc) {
        if (p.TH == kThreads && p.R == 2)
            launch(norm_nhwc_one_kernel<T, V, 2, kThreads>, grid, block, s, a);
        else if (p.TH == kThreads)
            launch(norm_nhwc_one_kernel<T, V, 4, kThreads>, grid, block, s, a);
        else if (p.R == 4)
            launch(norm_nhwc_one_kernel<T, V, 4, kWide>, grid, block, s, a);
        else
            launch(norm_nhwc_one_kernel<T, V, 8, kWide>, grid, block, s, a);
    } else if constexpr (V == 1 || V * sizeof(T) == 16) {  // NCHW takes these alone
        if (p.TH == kThreads && p.R == 2)
            launch(norm_nchw_one_kernel<T, V, 2, kThreads>, grid, block, s, a);
        else if (p.TH == kThreads)
            launch(norm_nchw_one_kernel<T, V, 4, kThreads>, grid, block, s, a);
        else
            launch(norm_nchw_one_kernel<T, V, 4, kWide>, grid, block, s, a);
    }
}

template <typename T, int V>
void forward_v(const GroupNorm& g, const Plan& p, const GnArgs& a, hipStream_t s) {
    if (p.form == kOne) {
        one_v<T, V>(g, p, a, s);
        return;
    }
    const dim3 grid((unsigned)p.grid), block(p.TH), groups((unsigned)(g.B * g.G));
    if (g.nhwc) {
        const size_t lds = 4 * ((size_t)a.bands() * a.C + a.G);
        if (a.G > p.TH) launch_lds(stats_nhwc_kernel<T, V, true>, grid, block, lds, s, a);
        else launch_lds(stats_nhwc_kernel<T, V, false>, grid, block, lds, s, a);
        if (p.join) {
            launch(norm_join_kernel, groups, dim3(64), s, a, p.pieces);
            launch(apply_nhwc_kernel<T, V, false>, grid, block, s, a);
        } else {
            launch(apply_nhwc_kernel<T, V, true>, grid, block, s, a);
        }
    } else if constexpr (V == 1 || V * sizeof(T) == 16) {
        launch(stats_nchw_kernel<T, V>, grid, block, s, a);
        if (p.join) {
            launch(norm_join_kernel, groups, dim3(64), s, a, p.pieces * a.n);
            launch(apply_nchw_kernel<T, V, false>, grid, block, s, a);
        } else {
            launch(apply_nchw_kernel<T, V, true>, grid, block, s, a);
        }
    }
}

template <typename T>
void forward_t(const GroupNorm& g, const Plan& p, const GnArgs& a, hipStream_t s) {
    if (p.form == kPlain) {
        launch(norm_plain_kernel<T>, dim3((unsigned)(g.B * g.G)), dim3(kThreads), s, a);
        return;
    }
    constexpr int kMost = 16 / sizeof(T);
    if (p.V == kMost) forward_v<T, kMost>(g, p, a, s);
    else if (p.V == kMost / 2) forward_v<T, kMost / 2>(g, p, a, s);
    else if (p.V == 1) forward_v<T, 1>(g, p, a, s);
    else if constexpr (sizeof(T) == 2) forward_v<T, 2>(g, p, a, s);
}

// extra: workgroups of the last launch that write the parameters' gradients.
template <typename T, int V>
void backward_v(const GroupNorm& g, const Plan& p, const GnArgs& a, int extra, hipStream_t s) {
    const dim3 grid((unsigned)p.grid), block(p.TH);
    const dim3 joins((unsigned)(g.B * g.G)), last((unsigned)(p.grid + extra));
    if (!g.nhwc) {
        if constexpr (V == 1 || V * sizeof(T) == 16) {
            launch(sums_nchw_kernel<T, V>, grid, block, s, a);
            launch(sums_join_kernel, joins, dim3(kThreads), s, a);
            launch(dx_nchw_kernel<T, V>, last, block, s, a);
        }
    } else {
        launch_lds(sums_nhwc_kernel<T, V>, grid, block, 8 * a.bands() * a.C, s, a);
        launch(sums_join_kernel, joins, dim3(kThreads), s, a);
        launch(dx_nhwc_kernel<T, V>, last, block, s, a);
    }
}

template <typename T>
void backward_t(const GroupNorm& g, const Plan& p, const GnArgs& a, int extra, hipStream_t s) {
    if (p.form == kPlain) {
        launch(sums_plain_kernel<T>, dim3((unsigned)(g.B * g.C)), dim3(kThreads), s, a);
        launch(sums_join_kernel, dim3((unsigned)(g.B * g.G)), dim3(kThreads), s, a);
        launch(dx_plain_kernel<T>, dim3((unsigned)(a.grid + extra)), dim3(kThreads), s, a);
        return;
    }
    constexpr int kMost = 16 / sizeof(T);
    if (p.V == kMost) backward_v<T, kMost>(g, p, a, extra, s);
    else if (p.V == kMost / 2) backward_v<T, kMost / 2>(g, p, a, extra, s);
    else if (p.V == 1) backward_v<T, 1>(g, p, a, extra, s);
    else if constexpr (sizeof(T) == 2) backward_v<T, 2>(g, p, a, extra, s);
}

__global__ __launch_bounds__(kThreads) void zero_params_kernel(GnArgs a) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.C) return;
    store_param(a.dbeta, a.params, c, 0.0f);
    store_param(a.dgamma, a.params, c, 0.0f);
}

}  // namespace

// The vector length, and with it the pieces, follows the alignment of the
// call's tensors; the sizes below cover every alignment.
GroupNormLaunch group_norm_launch(const GroupNorm& g, bool backward, int cus) {
    GroupNormLaunch most{0, 0};
    if (g.B == 0 || g.P == 0) return most;
    auto add = [&](int64_t grid, int block) {
        most.threads = std::max(most.threads, grid * block);
        most.block = std::max(most.block, block);
    };
    for (uintptr_t align = 16; align >= 2; align /= 2) {
        const void* at = reinterpret_cast<const void*>(align);
        const Plan p = plan_of(g, &at, 1, backward, cus);
        const int64_t groups = (int64_t)g.B * g.G;
        if (p.form != kPlain) add(p.grid + (backward ? extra_of(g) : 0), p.TH);
        else if (backward) add(std::max<int64_t>((int64_t)g.B * g.C, plain_grid(g) + extra_of(g)),
                               kThreads);
        if (backward || p.form == kPlain) add(groups, kThreads);
        else if (p.join) add(groups, 64);
    }
    return most;
}

int64_t group_norm_ws(const GroupNorm& g, int cus) {
    int64_t most = 0;
    if (g.B == 0 || g.P == 0) return 0;
    for (uintptr_t align = 16; align >= 2; align /= 2) {
        const void* at = reinterpret_cast<const void*>(align);
        const Plan p = plan_of(g, &at, 1, false, cus);
        if (p.form == kPieces)
            most = std::max(most, 12 * (int64_t)g.B * p.pieces * (g.nhwc ? g.G : g.C));
    }
    return most;
}

hipError_t launch_group_norm(const GroupNorm& g, void* y, float* mean, float* rstd, void* ws,
                             int cus, hipStream_t s) {
    if (g.B == 0 || g.P == 0) return hipSuccess;
    const void* ptrs[] = {g.x, y};
    const Plan p = plan_of(g, ptrs, 2, false, cus);
    GnArgs a = args_of(g, p);
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.part = static_cast<float*>(ws);
    if (g.dtype == kF16) forward_t<_Float16>(g, p, a, s);
    else if (g.dtype == kBF16) forward_t<__bf16>(g, p, a, s);
    else forward_t<float>(g, p, a, s);
    return hipGetLastError();
}

int64_t group_norm_bwd_ws(const GroupNorm& g, int cus) {
    int64_t most = 1;
    if (g.B == 0 || g.P == 0) return 0;
    for (uintptr_t align = 16; align >= 2; align /= 2) {
        const void* at = reinterpret_cast<const void*>(align);
        const Plan p = plan_of(g, &at, 1, true, cus);
        most = std::max(most, (int64_t)std::max(p.pieces, 1));
    }
    return 8 * (int64_t)g.B * g.G + 8 * (int64_t)g.B * (most + 1) * g.C;
}

hipError_t launch_group_norm_bwd(const GroupNorm& g, const void* dy, const float* mean,
                                 const float* rstd, void* dx, void* dgamma, void* dbeta, void* ws,
                                 int cus, hipStream_t s) {
    const void* ptrs[] = {g.x, dy, dx};
    const Plan p = g.B == 0 || g.P == 0 ? Plan{} : plan_of(g, ptrs, 3, true, cus);
    GnArgs a = args_of(g, p);
    a.dy = dy;
    a.y = dx;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    if (g.B == 0 || g.P == 0) {
        if (dgamma != nullptr)
            launch(zero_params_kernel, dim3((unsigned)div_up(g.C, kThreads)), dim3(kThreads), s,
                   a);
        return hipGetLastError();
    }
    if (p.form == kPlain) a.grid = plain_grid(g);
    a.sums = static_cast<float*>(ws);
    a.part = a.sums + 2 * (int64_t)g.B * g.G;
    const int extra = dgamma != nullptr ? extra_of(g) : 0;
    if (g.dtype == kF16) backward_t<_Float16>(g, p, a, extra, s);
    else if (g.dtype == kBF16) backward_t<__bf16>(g, p, a, extra, s);
    else backward_t<float>(g, p, a, extra, s);
    return hipGetLastError();
}

}  // namespace nova
