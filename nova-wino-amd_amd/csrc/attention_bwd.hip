// Gradients of attention (attention_fwd.hip). With the forward's row
// statistics the probabilities p_ij = exp2(c q_i . k_j - lse_i) come back from
// one product, and
//
//   dv_j = sum_i p_ij do_i                     dp_ij = do_i . v_j
//   ds_ij = p_ij (dp_ij - delta_i)             delta_i = sum_j p_ij dp_ij = do_i . o_i
//   dq_i = scale sum_j ds_ij k_j               dk_j = scale sum_i ds_ij q_i
//
// Two kernels, neither with atomics: one owns query rows and walks the keys
// (dq, delta), one owns keys and walks the query rows of every head, and every
// sequence, that reads them (dk, dv). Each holds its own rows one per lane, as
// the forward does, so p and ds leave one product as the operand of the next.
//
// In float16, ds can lie far below the type's smallest normal number, and so
// can p: p enters its product times 2^10, and ds times a power of two that
// each lane keeps for its row or key, moved (with the sums so far) only when a
// tile's largest value would leave the type's range. bfloat16 has float32's
// range and needs neither.
//
// What bounds them: the vector work on p and ds beside the products, at one or
// two waves a SIMD (a row's q, do and dq, or a key's k, v, dk and dv fill the
// registers). 3 x 12 heads x 1000 rows of 80, 333 keys, bfloat16: dq 24 us, dk
// and dv 36 us, the join 6 us. One owner of a row or key with both walks
// computes p and ds twice, and needs no atomics, whose order would change
// results.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace nova {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;
constexpr int kQueryTile = 64;  // query rows per tile of the kernel that owns keys
constexpr int kKeys = 128;      // keys of its workgroup

struct BwdArgs {
    const uint16_t *q, *k, *v, *out, *rest, *go;
    const uint8_t* mask;
    const float* lse;
    float* delta;  // [B][H][Lq]
    uint16_t *dq, *dk, *dv;
    float* part;  // [splits][2][Bk][Lk][KV][D] float32 sums of dk and dv, or null
    int64_t qs[3], ks[3], vs[3], mask_stride;
    int B, Bk, Lq, Lk, H, KV, group, D;
    int qblocks, nq;                         // dq: workgroups
    int kblocks, splits, per, units;         // dk, dv
    int nk;
    int qvec, kvec, vvec, ovec;
    float c, scale;       // the scores' factor (see score_scale); |scale|
    unsigned flip, live;  // sign bits of the queries, set where scale < 0; 0 for a scale of 0
    int fine;             // p and ds enter as two terms each
};

// A lane's power of two for ds in float16 and what follows from a change.
struct Range {
    float f = 0.0f;  // values go into the product times f; 0: none seen yet
    // largest: the tile's largest |ds| of the lane's row. Returns what the sums
    // so far have to be multiplied with.
    __device__ __forceinline__ float fit(float largest) {
        if (!(largest * f > 32768.0f || (f == 0.0f && largest > 0.0f))) return 1.0f;
        const float nf = __builtin_ldexpf(1.0f, half_range(largest));
        const float r = f == 0.0f ? 1.0f : nf / f;  // both powers of two
        f = nf;
        return r;
    }
};

// What packing x * f into p dropped, packed in its place.
template <typename T>
__device__ __forceinline__ void rests(unsigned (&p)[2][8], const f16v (&x)[2], float f) {
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int r = 0; r < 16; r += 2)
            p[b][r / 2] = T::pack(x[b][r] * f - T::lo(p[b][r / 2]),
                                  x[b][r + 1] * f - T::hi(p[b][r / 2]));
}

template <typename T, int DK, int DV>
__global__ __launch_bounds__(kThreads, DV <= 3 ? 2 : 1) void attention_dq_kernel(BwdArgs a) {
    typedef Tile<64 * ((DV + 1) / 2)> KV;
    __shared__ __attribute__((aligned(1024))) uint16_t kt[2][KV::kElems], vt[2][KV::kElems];
    __shared__ uint64_t bits[kMaskTiles];

    const int id = xcd_remap(blockIdx.x, a.nq);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rest = id;
    const int qb = rest % a.qblocks;
    rest /= a.qblocks;
    const int h = rest % a.H, b = rest / a.H;
    const int kvh = h / a.group, bk = a.Bk == 1 ? 0 : b;
    const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
    const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
    const typename KV::Fill kfill(tid, a.ks[1], a.D), vfill(tid, a.vs[1], a.D);
    const typename KV::Lane at(lane);

    const int row = qb * kRows + wave * 32 + (lane & 31);
    const bool live = row < a.Lq;
    const int64_t srow = ((int64_t)b * a.H + h) * a.Lq + row;
    const int64_t orow = (((int64_t)b * a.Lq + row) * a.H + h) * a.D;
    u4 qf[DK], gf[DK];
    float delta = 0.0f, lse = INFINITY;
    {
        const int64_t i = min(row, a.Lq - 1);
        const int64_t orow = (((int64_t)b * a.Lq + i) * a.H + h) * a.D;
        load_row<DK>(a.q + b * a.qs[0] + h * a.qs[2] + i * a.qs[1], live, half, a.D, a.qvec, qf);
        load_row<DK>(a.go + orow, live, half, a.D, a.ovec, gf);
#pragma unroll
        for (int s = 0; s < DK; s++) qf[s] = (qf[s] & a.live) ^ a.flip;
        if (a.out) {  // else one tile holds every key
            u4 of[DK], rf[DK];
            load_row<DK>(a.out + orow, live, half, a.D, a.ovec, of);
            if (a.rest) load_row<DK>(a.rest + orow, live, half, a.D, a.ovec, rf);
#pragma unroll
            for (int s = 0; s < DK; s++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const unsigned r = a.rest ? rf[s][j] : 0u;
                    delta = __builtin_fmaf(T::lo(gf[s][j]), T::lo(of[s][j]) + T::lo(r), delta);
                    delta = __builtin_fmaf(T::hi(gf[s][j]), T::hi(of[s][j]) + T::hi(r), delta);
                }
        }
        if (live) lse = a.lse[srow];
    }
    delta = add_halves(delta);

    f16v acc[DV];
#pragma unroll
    for (int d = 0; d < DV; d++) acc[d] = f16v{};
    Range range;

    KeyTiles tiles(0, (a.Lk + kKeyTile - 1) / kKeyTile, a.Lk,
                   a.mask ? a.mask + b * a.mask_stride : nullptr, bits, kWaves);
    auto fill = [&](int buf, int t, uint64_t keep) {
        const int64_t j = (int64_t)t * kKeyTile;
        kfill(kt[buf], kp + j * a.ks[1], a.ks[1], keep, a.D, a.kvec, tid);
        vfill(vt[buf], vp + j * a.vs[1], a.vs[1], keep, a.D, a.vvec, tid);
    };
    uint64_t now, next;
    int t = tiles.next(&now), buf = 0;
    if (now != 0) fill(0, t, now);
    for (; now != 0; now = next, buf ^= 1) {
        wait_vmcnt<0>();
        lds_barrier();
        t = tiles.next(&next);
        if (next != 0) fill(buf ^ 1, t, next);
        {
            f16v s[2], g[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                s[kb] = g[kb] = f16v{};
#pragma unroll
                for (int st = 0; st < DK; st++) {
                    s[kb] = T::mfma(KV::rows(kt[buf], at, 32 * kb, st), qf[st], s[kb]);
                    g[kb] = T::mfma(KV::rows(vt[buf], at, 32 * kb, st), gf[st], g[kb]);
                }
            }
            const bool full = now == ~0ull;
            const uint64_t mine = now >> (4 * half);
            float own = 0.0f;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.c, -lse));
                    if (!full && !((mine >> (32 * kb + acc_row(r))) & 1)) s[kb][r] = 0.0f;
                    own = __builtin_fmaf(s[kb][r], g[kb][r], own);
                }
            // one tile holds every key: delta without the rounding of o
            if (!a.out) delta = add_halves(own);
            float top = 0.0f;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[kb][r] *= g[kb][r] - delta;
                    top = fmaxf(top, fabsf(s[kb][r]));
                }
            float f = 1.0f;
            if (T::kHalf) {
                const float fix = range.fit(max_halves(top));
                f = range.f;
                if (__any(fix != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DV; d++) acc[d] *= fix;
                }
            }
            unsigned p[2][8];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r += 2)
                    p[kb][r / 2] = T::pack(s[kb][r] * f, s[kb][r + 1] * f);
            auto products = [&] {
#pragma unroll
                for (int d = 0; d < DV; d++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const unsigned* pp = &p[x >> 1][4 * (x & 1)];
                        acc[d] = T::mfma(KV::turned(kt[buf], at, 16 * x, d),
                                         u4{pp[0], pp[1], pp[2], pp[3]}, acc[d]);
                    }
            };
            products();
            if (a.fine) {
                rests<T>(p, s, f);
                products();
            }
        }
    }
    if (!live) return;
    if (half == 0) a.delta[srow] = delta;
    float f = a.flip ? -a.scale : a.scale;
    if (T::kHalf) f = range.f == 0.0f ? 0.0f : f / range.f;
    uint16_t* p = a.dq + orow;
    store_row<T, DV>(p, nullptr, acc, f, half, a.D);
}

// A workgroup owns 128 keys of one KV head, one per lane of its waves, and walks
// its range of the query tiles: every tile of every query head that reads the KV
// head, of every sequence that reads these keys. The next tile's rows go to LDS
// while the current one is worked on.
template <typename T, int DK, int DV, bool FINE>
__global__ __launch_bounds__(kThreads, DV <= 2 && !FINE ? 2 : 1) void attention_dkv_kernel(BwdArgs a) {
    typedef Tile<64 * ((DV + 1) / 2)> Q;
    __shared__ __attribute__((aligned(1024))) uint16_t qt[2][Q::kElems], gt[2][Q::kElems];
    __shared__ __attribute__((aligned(16))) float slse[2][kQueryTile], sdelta[2][kQueryTile];

    const int id = xcd_remap(blockIdx.x, a.nk);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rest = id;
    const int kblock = rest % a.kblocks;
    rest /= a.kblocks;
    const int split = rest % a.splits;
    rest /= a.splits;
    const int kvh = rest % a.KV, bk = rest / a.KV;
    const typename Q::Lane at(lane);
    const int64_t gstride = (int64_t)a.H * a.D;
    const typename Q::Fill qfill(tid, a.qs[1], a.D), gfill(tid, gstride, a.D);

    const int key = kblock * kKeys + wave * 32 + (lane & 31);
    const bool inside = key < a.Lk;
    u4 kf[DK], vf[DK];
    {
        // a key that no sequence keeps may hold anything: it is read as zeros
        bool used = inside;
        if (a.mask && inside) {
            used = false;
            if (a.Bk == 1)
                for (int b = 0; b < a.B; b++) used |= a.mask[b * a.mask_stride + key] != 0;
            else
                used = a.mask[bk * a.mask_stride + key] != 0;
        }
        const int64_t j = min(key, a.Lk - 1);
        load_row<DK>(a.k + bk * a.ks[0] + kvh * a.ks[2] + j * a.ks[1], used, half, a.D, a.kvec,
                     kf);
        load_row<DK>(a.v + bk * a.vs[0] + kvh * a.vs[2] + j * a.vs[1], used, half, a.D, a.vvec,
                     vf);
        // the scale's sign (or a scale of 0), which the other kernels give the queries
#pragma unroll
        for (int s = 0; s < DK; s++) kf[s] = (kf[s] & a.live) ^ a.flip;
    }

    f16v dk[DV], dv[DV];
#pragma unroll
    for (int d = 0; d < DV; d++) dk[d] = dv[d] = f16v{};
    Range range;

    const int u0 = split * a.per, u1 = min(a.units, u0 + a.per);
    const int nqt = (a.Lq + kQueryTile - 1) / kQueryTile;
    float nlse = 0.0f, ndelta = 0.0f;  // of row tid of the tile on its way
    auto fetch = [&](const QueryTile& p, int buf) {
        const int row0 = p.tile * kQueryTile, h = kvh * a.group + p.head, b = p.seq;
        const int n = a.Lq - row0;
        const uint64_t rows = n >= kQueryTile ? ~0ull : (1ull << n) - 1;
        qfill(qt[buf], a.q + b * a.qs[0] + h * a.qs[2] + row0 * a.qs[1], a.qs[1], rows, a.D,
              a.qvec, tid);
        gfill(gt[buf], a.go + (((int64_t)b * a.Lq + row0) * a.H + h) * a.D, gstride, rows, a.D,
              a.ovec, tid);
        nlse = INFINITY;
        ndelta = 0.0f;
        if (tid < min(n, kQueryTile)) {
            const int64_t srow = ((int64_t)b * a.H + h) * a.Lq + row0 + tid;
            nlse = a.lse[srow];
            ndelta = a.delta[srow];
        }
    };
    auto put_stats = [&](int buf) {
        if (tid < kQueryTile) {
            slse[buf][tid] = nlse;
            sdelta[buf][tid] = ndelta;
        }
    };
    int buf = 0;
    QueryTile now(u0, nqt, a.group, a.Bk == 1 ? 0 : bk), after = now;
    if (u0 < u1) {
        fetch(now, 0);
        put_stats(0);
    }
    for (int u = u0; u < u1; u++, buf ^= 1) {
        const bool keep =
            inside && (a.mask == nullptr || a.mask[now.seq * a.mask_stride + key] != 0);
        after.next(nqt, a.group);
        wait_vmcnt<0>();
        lds_barrier();
        if (u + 1 < u1) fetch(after, buf ^ 1);
        now = after;

        f16v s[2], g[2];
#pragma unroll
        for (int rb = 0; rb < 2; rb++) {
            s[rb] = g[rb] = f16v{};
#pragma unroll
            for (int st = 0; st < DK; st++) {
                s[rb] = T::mfma(Q::rows(qt[buf], at, 32 * rb, st), kf[st], s[rb]);
                g[rb] = T::mfma(Q::rows(gt[buf], at, 32 * rb, st), vf[st], g[rb]);
            }
        }
        constexpr float kUp = T::kHalf ? 10.0f : 0.0f;  // p times 2^10
        unsigned p[2][8];
        float top = 0.0f;
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int i = 32 * rb + acc_row(r) + 4 * half;
                const f4 ls = *reinterpret_cast<const f4*>(slse[buf] + i);
                const f4 de = *reinterpret_cast<const f4*>(sdelta[buf] + i);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(s[rb][r + e], a.c, kUp - ls[e]));
                    if (!keep) x = 0.0f;
                    s[rb][r + e] = x;
                    float y = x * (g[rb][r + e] - de[e]);
                    if (!keep) y = 0.0f;
                    g[rb][r + e] = y;
                    top = fmaxf(top, fabsf(y));
                }
                p[rb][r / 2] = T::pack(s[rb][r], s[rb][r + 1]);
                p[rb][r / 2 + 1] = T::pack(s[rb][r + 2], s[rb][r + 3]);
            }
        auto products = [&](const uint16_t* t, f16v(&sum)[DV]) {
#pragma unroll
            for (int d = 0; d < DV; d++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const unsigned* pp = &p[x >> 1][4 * (x & 1)];
                    sum[d] = T::mfma(Q::turned(t, at, 16 * x, d),
                                     u4{pp[0], pp[1], pp[2], pp[3]}, sum[d]);
                }
        };
        products(gt[buf], dv);
        if (FINE) {
            rests<T>(p, s, 1.0f);
            products(gt[buf], dv);
        }
        float f = 1.0f;
        if (T::kHalf) {
            const float fix = range.fit(max_halves(top));
            f = range.f;
            if (__any(fix != 1.0f)) {
#pragma unroll
                for (int d = 0; d < DV; d++) dk[d] *= fix;
            }
        }
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int r = 0; r < 16; r += 2)
                p[rb][r / 2] = T::pack(g[rb][r] * f, g[rb][r + 1] * f);
        products(qt[buf], dk);
        if (FINE) {
            rests<T>(p, g, f);
            products(qt[buf], dk);
        }
        if (u + 1 < u1) put_stats(buf ^ 1);
    }

    if (!inside) return;
    float fk = a.flip ? -a.scale : a.scale, fv = 1.0f;
    if (T::kHalf) {
        fk = range.f == 0.0f ? 0.0f : fk / range.f * 0x1p-10f;
        fv = 0x1p-10f;
    }
    const int64_t krow = (((int64_t)bk * a.Lk + key) * a.KV + kvh) * a.D;
    const int64_t all = (int64_t)a.Bk * a.Lk * a.KV * a.D;
#pragma unroll
    for (int d = 0; d < DV; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int e = 32 * d + acc_row(r) + 4 * half;
            if (e >= a.D) continue;
            const float x = dk[d][r] * fk, y = dv[d][r] * fv;
            if (a.part) {
                a.part[2 * split * all + krow + e] = x;
                a.part[(2 * split + 1) * all + krow + e] = y;
            } else {
                a.dk[krow + e] = (uint16_t)T::pack(x, 0.0f);
                a.dv[krow + e] = (uint16_t)T::pack(y, 0.0f);
            }
        }
}

// Adds the ranges' float32 sums of dk and dv in their order and rounds once:
// 4 to 6 us, a launch and two trips to memory.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_dkv_join_kernel(const float* part,
                                                                      uint16_t* dk, uint16_t* dv,
                                                                      int64_t all, int splits) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= 2 * all) return;
    float x = 0.0f;
#pragma unroll 8
    for (int s = 0; s < splits; s++) x += part[2 * s * all + i];
    const uint16_t r = (uint16_t)T::pack(x, 0.0f);
    if (i < all) dk[i] = r;
    else dv[i - all] = r;
}

template <typename T>
hipError_t launch_join(const float* part, uint16_t* dk, uint16_t* dv, int64_t all, int splits,
                       hipStream_t s) {
    launch(attention_dkv_join_kernel<T>, dim3((unsigned)((2 * all + kThreads - 1) / kThreads)),
           dim3(kThreads), s, part, dk, dv, all, splits);
    return hipGetLastError();
}

template <typename T, int DK, int DV>
void launch_pair(const BwdArgs& f, hipStream_t s) {
    if (f.nq > 0)
        launch(attention_dq_kernel<T, DK, DV>, dim3((unsigned)f.nq), dim3(kThreads), s, f);
    if (f.nk > 0 && f.fine)
        launch(attention_dkv_kernel<T, DK, DV, true>, dim3((unsigned)f.nk), dim3(kThreads), s, f);
    else if (f.nk > 0)
        launch(attention_dkv_kernel<T, DK, DV, false>, dim3((unsigned)f.nk), dim3(kThreads), s,
               f);
}

template <typename T>
hipError_t launch_all(const BwdArgs& f, hipStream_t s) {
    const int dk = (f.D + 15) / 16;
    if (dk <= 2) launch_pair<T, 2, 1>(f, s);
    else if (dk <= 3) launch_pair<T, 3, 2>(f, s);
    else if (dk <= 4) launch_pair<T, 4, 2>(f, s);
    else if (dk <= 5) launch_pair<T, 5, 3>(f, s);
    else if (dk <= 6) launch_pair<T, 6, 3>(f, s);
    else if (dk <= 8) launch_pair<T, 8, 4>(f, s);
    else if (dk <= 10) launch_pair<T, 10, 5>(f, s);
    else launch_pair<T, 16, 8>(f, s);
    if (f.part)
        return launch_join<T>(f.part, f.dk, f.dv, (int64_t)f.Bk * f.Lk * f.KV * f.D, f.splits, s);
    return hipGetLastError();
}

}  // namespace

// Bytes of delta in front of the workspace, in whole 16s.
static int64_t delta_bytes(const Attention& a) {
    return ((int64_t)4 * a.B * a.H * a.Lq + 15) / 16 * 16;
}

// The short form: the keys that a workgroup's LDS holds; keys that sequences
// share under a mask may hold anything where another sequence keeps them, which
// the long form's walks tell apart. The short form against the tiles, backward
// alone, us: 64 heads of 40, 4096 rows, 77 keys 50 | 80; 64 heads of 80, 1024 rows,
// 128 keys 41 | 54; 16 heads of 160, 4096 rows, 96 keys 84 | 96 in bfloat16. In
// float16, where both keep some of that size's values in scratch, 114 | 108; 64
// heads of 160, 1024 rows, 77 keys 110 | 105, 60 keys 77 | 85, 8 heads 39 | 54. The
// forward is 6 us faster without the rest that it writes for the tiles, so that
// those steps are even: 133 | 134, and 137 | 137 with 96 keys.
//
// Few rows in the whole call take the long form with p and ds as two terms each.
// One rounding of p and ds makes a gradient's error 1.42 times that of its own
// last rounding for any number of rows; two terms, 1.04. What few rows change is
// the spread: few p and ds hold most of a gradient, and their luck decides.
// Largest of 24 calls, one term | two: 1 row 2.4 | 1.0, 64 rows 1.64 | 1.07, 512
// rows 1.53 | 1.06, 1024 rows 1.50. The price, forward and backward, us, for 512
// rows of 64 channels: 77 keys, one head 23 | 32, 64 heads 15 | 27, 512 heads 19 |
// 42; 333 keys, one head 43 | 46; 1500 keys, 64 heads 100 | 112 (a step's host part
// is some 65 outside of a graph).
static bool few_rows(const Attention& a) { return (int64_t)a.B * a.H * a.Lq <= 512; }

static bool short_bwd(const Attention& a) {
    return !few_rows(a) && a.Lk >= 1 && a.Lq >= 1 && a.Bk >= 1 && a.D <= kShortChannels &&
           a.Lk <= (a.D <= 16 * kShortDeep ? kShortKeys : 96) &&
           (a.mask == nullptr || a.Bk == a.B);
}

bool attention_uses_rest(const Attention& a) { return !short_bwd(a) && a.Lk > kKeyTile; }

AttentionBwdPlan attention_bwd_plan(const Attention& a, int cus) {
    AttentionBwdPlan p{};
    p.whole = short_bwd(a);
    p.rows = p.whole ? (a.Lk <= 64 ? 64 : a.Lk <= 96 ? 96 : 128) : kQueryTile;
    p.kblocks = p.whole ? 1 : (a.Lk + kKeys - 1) / kKeys;
    p.units = (a.B / std::max(a.Bk, 1)) * (a.H / a.KV) * ((a.Lq + p.rows - 1) / p.rows);
    const int64_t wgs = (int64_t)a.Bk * a.KV * p.kblocks;
    // As many ranges of rows as give every CU a workgroup (the short form: two):
    // fewer leave CUs idle (3 x 12 heads of 80, 1000 rows, 333 keys: 44 us with
    // the join, half as many 54), more cost the join what they gain (128 heads of
    // 64, 256 rows, 256 keys: 23 us, twice as many 43).
    const int room = (p.whole ? 2 : 1) * cus;
    // Down to one tile a range, where the join's launch does not cost more than
    // that gains (16 heads of 40, 1024 rows, 77 keys: 11 ranges 17 us with the
    // join, 5 ranges 23; 40 heads of 64, 256 rows: 3 ranges 20, one 18).
    const int64_t most = p.units >= 6 ? p.units : p.units / 2;
    const int64_t n = std::max<int64_t>(
        1, std::min({room / std::max<int64_t>(wgs, 1), most, (int64_t)64}));
    p.per = (int)std::max<int64_t>(1, (p.units + n - 1) / n);
    p.splits = std::max(1, (p.units + p.per - 1) / p.per);
    if (a.Lk == 0) p.splits = 1;  // no sums to join
    p.ws_bytes = p.whole ? 0 : delta_bytes(a);
    if (p.splits > 1) p.ws_bytes += 8 * (int64_t)p.splits * a.Bk * a.Lk * a.KV * a.D;
    return p;
}

hipError_t launch_attention_bwd(const Attention& a, const AttentionBwdPlan& plan,
                                const uint16_t* out, const uint16_t* rest, const float* lse,
                                const uint16_t* go, uint16_t* dq, uint16_t* dk, uint16_t* dv,
                                void* ws, hipStream_t s) {
    if (plan.whole) {
        float* part = plan.splits > 1 ? static_cast<float*>(ws) : nullptr;
        const hipError_t e = launch_attention_short_bwd(a, plan, lse, go, dq, dk, dv, part, s);
        if (e != hipSuccess || part == nullptr) return e;
        const int64_t all = (int64_t)a.Bk * a.Lk * a.KV * a.D;
        return a.bf16 ? launch_join<BF16>(part, dk, dv, all, plan.splits, s)
                      : launch_join<F16>(part, dk, dv, all, plan.splits, s);
    }
    BwdArgs f{};
    f.q = a.q;
    f.k = a.k;
    f.v = a.v;
    if (attention_uses_rest(a)) {
        f.out = out;
        f.rest = rest;
    }
    f.go = go;
    f.mask = a.mask;
    f.lse = lse;
    f.delta = static_cast<float*>(ws);
    f.dq = dq;
    f.dk = dk;
    f.dv = dv;
    std::copy(a.qs, a.qs + 3, f.qs);
    std::copy(a.ks, a.ks + 3, f.ks);
    std::copy(a.vs, a.vs + 3, f.vs);
    f.mask_stride = a.mask_stride;
    f.B = a.B;
    f.Bk = a.Bk;
    f.Lq = a.Lq;
    f.Lk = a.Lk;
    f.H = a.H;
    f.KV = a.KV;
    f.group = a.H / a.KV;
    f.D = a.D;
    f.qblocks = (a.Lq + kRows - 1) / kRows;
    f.nq = a.B * a.H * f.qblocks;
    f.kblocks = plan.kblocks;
    f.splits = plan.splits;
    f.per = plan.per;
    f.units = plan.units;
    f.nk = a.Bk * a.KV * plan.kblocks * plan.splits;
    f.qvec = chunked(a.q, a.qs, a.D) && close_rows(a.qs[1]);
    f.kvec = chunked(a.k, a.ks, a.D) && close_rows(a.ks[1]);
    f.vvec = chunked(a.v, a.vs, a.D) && close_rows(a.vs[1]);
    const int64_t os[3] = {a.D, a.D, a.D};
    f.ovec = chunked(out, os, a.D) && chunked(go, os, a.D) && chunked(rest, os, a.D) &&
             close_rows((int64_t)a.H * a.D);
    f.scale = std::fabs(a.scale);
    f.c = score_scale(a);
    f.flip = a.scale < 0 ? 0x80008000u : 0u;
    f.live = a.scale != 0 ? ~0u : 0u;
    f.fine = few_rows(a);
    if (plan.splits > 1)
        f.part = reinterpret_cast<float*>(static_cast<char*>(ws) + delta_bytes(a));
    return a.bf16 ? launch_all<BF16>(f, s) : launch_all<F16>(f, s);
}

}  // namespace nova
