// Attention of queries to the keys and values of another sequence:
//
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j)  over the kept keys j
//
// in one pass over the keys with the running maximum and sum of each row.
//
// A wave holds 32 query rows, one per lane (both lanes l and l + 32 hold row
// l). S^T = K Q^T puts the scores of a row into its lanes (32x32x16 MFMA, keys
// along the accumulators), so maximum, exp2 and sum run inside a lane with one
// exchange between the halves, and P^T is already the B operand of
// O^T = V^T P^T: Tile::turned reads V with the same order of keys. K and V
// tiles of 64 keys go from memory straight to LDS, the next pair while the
// current one is worked on.
// Scores, statistics and O are float32; P is rounded to the inputs' type for
// its product (values up to 1, where that type's spacing is the smallest
// relative to the row's largest).
// What bounds this kernel is the issue of its vector work (softmax) beside the
// matrix unit's: 4 x 16 heads x 4096 rows, 1024 keys of 128 channels in 195 us,
// 705 TFLOP/s; 2 x 64 heads x 1024 rows, 1024 keys of 64 in 55 us, 625 TFLOP/s.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace nova {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // query rows of a workgroup

struct FwdArgs {
    const uint16_t *q, *k, *v;
    const uint8_t* mask;
    uint16_t *out, *rest;
    float* lse;
    float* part;  // [splits][B][Lq][H][D] float32, or null: out is written
    float* plse;  // [splits][B][H][Lq]
    int64_t qs[3], ks[3], vs[3], mask_stride;
    int B, Bk, Lq, Lk, H, group, D;
    int qblocks, splits, per, n, pair;
    int qvec, kvec, vvec;  // rows in 16-byte chunks
    // The scores are c q . k, c > 0: the scale's sign goes into the queries
    // (flip: their sign bits), and a scale of 0 makes them zeros (live: 0).
    float c, lowest;  // lowest: see lowest_score
    unsigned flip, live;
};

// Channels at .. at + 3 of a dense float32 row of D, those that exist.
__device__ __forceinline__ void put_part(float* row, int at, int D, f4 v) {
    if ((D & 3) == 0) {  // rows then start on 16 bytes
        if (at < D) *reinterpret_cast<f4*>(row + at) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (at + e < D) row[at + e] = v[e];
    }
}

// A row's end: its sum from both halves, its statistic, its output (or, for a
// range of keys, its float32 part).
template <typename T, int DV>
__device__ __forceinline__ void finish_row(const FwdArgs& a, int b, int h, int split, int row,
                                           int half, float m, float l, const f16v (&o)[DV]) {
    l = add_halves(l);
    if (row >= a.Lq) return;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // no keys: 0; NaN stays
    const float stat = l == 0.0f ? INFINITY : m * a.c + __builtin_amdgcn_logf(l);
    const int64_t srow = ((int64_t)b * a.H + h) * a.Lq + row;
    if (a.part) {
        if (half == 0) a.plse[(int64_t)split * a.B * a.H * a.Lq + srow] = stat;
        float* p = a.part +
                   (((int64_t)split * a.B + b) * a.Lq + row) * a.H * a.D + (int64_t)h * a.D;
#pragma unroll
        for (int d = 0; d < DV; d++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                put_part(p, 32 * d + acc_row(r) + 4 * half, a.D,
                         f4{o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv,
                             o[d][r + 3] * inv});
        return;
    }
    if (a.lse && half == 0) a.lse[srow] = stat;
    uint16_t* p = a.out + (((int64_t)b * a.Lq + row) * a.H + h) * a.D;
    store_row<T, DV>(p, a.rest ? a.rest + (p - a.out) : nullptr, o, inv, half, a.D);
}

// Waves per SIMD that the registers leave room for: two up to 128 channels, so
// that one wave's products run under the other's softmax.
constexpr int waves_per_simd(int DV) { return DV <= 4 ? 2 : 1; }

template <typename T, int DK, int DV>
__global__ __launch_bounds__(kThreads, waves_per_simd(DV)) void attention_kernel(FwdArgs a) {
    typedef Tile<64 * ((DV + 1) / 2)> KV;
    __shared__ __attribute__((aligned(1024))) uint16_t kt[2][KV::kElems], vt[2][KV::kElems];
    __shared__ uint64_t bits[kMaskTiles];

    const int id = xcd_remap(blockIdx.x, a.n);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rest = id;
    const int qb = rest % a.qblocks;
    rest /= a.qblocks;
    const int split = rest % a.splits;
    rest /= a.splits;
    const int h = rest % a.H, b = rest / a.H;
    const int kvh = h / a.group, bk = a.Bk == 1 ? 0 : b;
    const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
    const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
    const typename KV::Fill kfill(tid, a.ks[1], a.D), vfill(tid, a.vs[1], a.D);
    const typename KV::Lane at(lane);

    const int row = qb * kRows + wave * 32 + (lane & 31);
    u4 qf[DK];
    {
        const uint16_t* qp = a.q + b * a.qs[0] + h * a.qs[2] + min(row, a.Lq - 1) * a.qs[1];
        load_row<DK>(qp, row < a.Lq, half, a.D, a.qvec, qf);
#pragma unroll
        for (int s = 0; s < DK; s++) qf[s] = (qf[s] & a.live) ^ a.flip;
    }

    f16v o[DV];
#pragma unroll
    for (int d = 0; d < DV; d++) o[d] = f16v{};
    float m = a.lowest, l = 0.0f;  // the row's maximum; this lane's part of its sum

    KeyTiles tiles(split * a.per,
                   min((a.Lk + kKeyTile - 1) / kKeyTile, split * a.per + a.per), a.Lk,
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

        f16v s[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            s[kb] = f16v{};
#pragma unroll
            for (int st = 0; st < DK; st++)
                s[kb] = T::mfma(KV::rows(kt[buf], at, 32 * kb, st), qf[st], s[kb]);
        }
        if (now != ~0ull) {
            const uint64_t mine = now >> (4 * half);
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!((mine >> (32 * kb + acc_row(r))) & 1)) s[kb][r] = -INFINITY;
        }
        float tm = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) tm = fmaxf(tm, s[kb][r]);
        const float mn = fmaxf(m, max_halves(tm));
        const float alpha = __builtin_amdgcn_exp2f((m - mn) * a.c), mc = mn * a.c;
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DV; d++) o[d] *= alpha;
        unsigned p[2][8];
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.c, -mc));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], a.c, -mc));
                l += x + y;
                p[kb][r / 2] = T::pack(x, y);
            }
#pragma unroll
        for (int d = 0; d < DV; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const unsigned* pp = &p[g >> 1][4 * (g & 1)];
                o[d] = T::mfma(KV::turned(vt[buf], at, 16 * g, d),
                               u4{pp[0], pp[1], pp[2], pp[3]}, o[d]);
            }
    }

    finish_row<T, DV>(a, b, h, split, row, half, m, l, o);
}

// N products, each of READS operand reads from LDS: the reads run kAhead products
// in front of the products, further than the compiler puts them by itself (two),
// which left each product waiting for its own.
constexpr int kAhead = 6;
template <int N, int READS>
__device__ __forceinline__ void ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead * READS, 0);
#pragma unroll
    for (int i = 0; i < N - kAhead; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, kAhead, 0);
    __builtin_amdgcn_sched_barrier(0);
}

// The same walk by two groups of four waves, half a tile apart: while one has its
// products (those of the last tile with V, then the next one's scores), the
// other has its softmax, so that a SIMD's two waves are never both at the matrix
// unit or both beside it. Left to themselves they are: the groups' barriers hold
// the phases apart. Slot n of a group runs from its n-th barrier on; the groups'
// loads of tile t + 1 start in slot 2 t, when the buffers they go to were last
// read a slot ago, and are waited for at the end of slot 2 t + 1.
// 4 x 16 heads x 4096 rows, 1024 keys of 128: 180 us, 765 TFLOP/s (one group's
// kernel above: 195). Products and vector work share half of their cycles now
// (before: a quarter). What bounds it is a SIMD's issue of the two: its
// registers hold two waves, and the softmax of one wave is as long as the
// products of the other. An order of the chunks in LDS without bank conflicts
// (they take half of its cycles in this one) measured the same time.
constexpr int kPairThreads = 2 * kThreads;
constexpr int kPairRows = 2 * kRows;

template <typename T, int DK, int DV>
__global__ __launch_bounds__(kPairThreads, 2) void attention_pair_kernel(FwdArgs a) {
    typedef Tile<64 * ((DV + 1) / 2)> KV;
    typedef typename KV::template FillBy<kPairThreads> Fill;
    __shared__ __attribute__((aligned(1024))) uint16_t kt[2][KV::kElems], vt[2][KV::kElems];
    __shared__ uint64_t bits[kMaskTiles];

    const int id = xcd_remap(blockIdx.x, a.n);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rest = id;
    const int qb = rest % a.qblocks;
    rest /= a.qblocks;
    const int split = rest % a.splits;
    rest /= a.splits;
    const int h = rest % a.H, b = rest / a.H;
    const int kvh = h / a.group, bk = a.Bk == 1 ? 0 : b;
    const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
    const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
    const Fill kfill(tid, a.ks[1], a.D), vfill(tid, a.vs[1], a.D);
    const typename KV::Lane at(lane);

    const int row = qb * kPairRows + wave * 32 + (lane & 31);
    u4 qf[DK];
    load_row<DK>(a.q + b * a.qs[0] + h * a.qs[2] + min(row, a.Lq - 1) * a.qs[1], row < a.Lq, half,
                 a.D, a.qvec, qf);
#pragma unroll
    for (int s = 0; s < DK; s++) qf[s] = (qf[s] & a.live) ^ a.flip;

    f16v o[DV];
#pragma unroll
    for (int d = 0; d < DV; d++) o[d] = f16v{};
    float m = a.lowest, l = 0.0f;
    KeyTiles tiles(split * a.per,
                   min((a.Lk + kKeyTile - 1) / kKeyTile, split * a.per + a.per), a.Lk,
                   a.mask ? a.mask + b * a.mask_stride : nullptr, bits, 2 * kWaves);

    unsigned p[2][8];
    f16v s[2];
    auto scores = [&](int buf) {
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            s[kb] = f16v{};
#pragma unroll
            for (int st = 0; st < DK; st++)
                s[kb] = T::mfma(KV::rows(kt[buf], at, 32 * kb, st), qf[st], s[kb]);
        }
        ahead<2 * DK, 1>();
    };
    auto values = [&](int buf) {
#pragma unroll
        for (int d = 0; d < DV; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const unsigned* pp = &p[g >> 1][4 * (g & 1)];
                o[d] = T::mfma(KV::turned(vt[buf], at, 16 * g, d),
                               u4{pp[0], pp[1], pp[2], pp[3]}, o[d]);
            }
        ahead<4 * DV, 2>();
    };
    auto softmax = [&](uint64_t now) {
        if (now != ~0ull) {
            const uint64_t mine = now >> (4 * half);
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!((mine >> (32 * kb + acc_row(r))) & 1)) s[kb][r] = -INFINITY;
        }
        float tm = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) tm = fmaxf(tm, s[kb][r]);
        const float mn = fmaxf(m, max_halves(tm));
        const float alpha = __builtin_amdgcn_exp2f((m - mn) * a.c), mc = mn * a.c;
        m = mn;
        l *= alpha;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.c, -mc));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], a.c, -mc));
                l += x + y;
                p[kb][r / 2] = T::pack(x, y);
            }
#pragma unroll
        for (int d = 0; d < DV; d++) o[d] *= alpha;
    };
    // the end of a slot; nothing crosses it
    auto slot = [&] {
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    // Tiles by number of the walk; kept keys of the tile whose scores are due
    // (now), of the one behind it (next).
    uint64_t now, next = 0;
    int t = tiles.next(&now), tv = t;
    if (now != 0) {
        const bool late = wave >= kWaves;
        auto load_k = [&](int buf, int tile, uint64_t keep) {
            kfill(kt[buf], kp + (int64_t)tile * kKeyTile * a.ks[1], a.ks[1], keep, a.D, a.kvec,
                  tid);
        };
        auto load_v = [&](int buf, int tile, uint64_t keep) {
            vfill(vt[buf], vp + (int64_t)tile * kKeyTile * a.vs[1], a.vs[1], keep, a.D, a.vvec,
                  tid);
        };
        load_k(0, t, now);
        wait_vmcnt<0>();
        int buf = 0;
        // the loads of slot 2 t: K of the next tile, V of this one
        auto load = [&] {
            tv = t;
            t = tiles.next(&next);
            load_v(buf, tv, now);
            if (next != 0) load_k(buf ^ 1, t, next);
        };
        slot();
        if (!late) {
            for (bool first = true;; first = false) {
                load();
                if (!first) values(buf ^ 1);
                scores(buf);
                slot();
                softmax(now);
                wait_vmcnt<0>();
                slot();
                buf ^= 1;
                if (next == 0) break;
                now = next;
            }
        } else {
            uint64_t before = 0;
            while (true) {
                load();
                if (before != 0) softmax(before);
                slot();
                if (before != 0) values(buf ^ 1);
                scores(buf);
                wait_vmcnt<0>();
                slot();
                before = now;
                buf ^= 1;
                if (next == 0) break;
                now = next;
            }
            softmax(before);
        }
        values(buf ^ 1);  // of the last tile
    }
    finish_row<T, DV>(a, b, h, split, row, half, m, l, o);
}

// Few rows (one new token of a decoder): the R rows that read one KV head stay
// in registers, LPK lanes hold one key (8 channels each) and every group of
// lanes walks its own keys with its own running maximum and sum; the groups,
// then the waves, are joined at the end. Keys that the mask drops are not
// read. The bytes of K and V bound it: 16 sequences x 16 heads, 1500 keys of 64
// in 17 us, 5.8 TB/s (some of it from the memory-side cache), and the join of
// the ranges of keys behind it takes 4 us.
template <typename T, int LPK, int R>
__global__ __launch_bounds__(kThreads) void attention_few_kernel(FwdArgs a) {
    constexpr int kKeys = 64 / LPK;  // keys of a wave's step
    constexpr int kDeep = R <= 2 ? 4 : 2;
    const int id = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int KV = a.H / a.group;
    int rest = id;
    const int split = rest % a.splits;
    rest /= a.splits;
    const int kvh = rest % KV, b = rest / KV;
    const int bk = a.Bk == 1 ? 0 : b;
    const int d = 8 * (lane % LPK), sub = lane / LPK;
    const int rows = a.group * a.Lq;  // row r: head kvh * group + r / Lq, query r % Lq
    const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
    const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
    const uint8_t* mp = a.mask ? a.mask + b * a.mask_stride : nullptr;

    float q[R][8], o[R][8], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        m[r] = a.lowest;
        l[r] = 0.0f;
        u4 x = {0, 0, 0, 0};
        if (r < rows) {
            const int h = kvh * a.group + r / a.Lq;
            x = (load_chunk(a.q + b * a.qs[0] + (int64_t)(r % a.Lq) * a.qs[1] + h * a.qs[2], d,
                            a.D, a.qvec) & a.live) ^ a.flip;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            q[r][2 * j] = T::lo(x[j]);
            q[r][2 * j + 1] = T::hi(x[j]);
            o[r][2 * j] = o[r][2 * j + 1] = 0.0f;
        }
    }

    const int j0 = split * a.per, j1 = min(a.Lk, j0 + a.per);
    for (int base = j0 + wave * kKeys; base < j1; base += kWaves * kKeys * kDeep) {
        u4 kr[kDeep], vr[kDeep];
        bool ok[kDeep];
#pragma unroll
        for (int u = 0; u < kDeep; u++) {
            const int j = base + u * kWaves * kKeys + sub;
            ok[u] = j < j1 && (mp == nullptr || mp[j] != 0);
            kr[u] = vr[u] = u4{0, 0, 0, 0};
            if (ok[u]) {
                kr[u] = load_chunk(kp + j * a.ks[1], d, a.D, a.kvec);
                vr[u] = load_chunk(vp + j * a.vs[1], d, a.D, a.vvec);
            }
        }
        float s[kDeep][R];
#pragma unroll
        for (int u = 0; u < kDeep; u++)
#pragma unroll
            for (int r = 0; r < R; r++) {
                float x = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x = __builtin_fmaf(q[r][2 * j], T::lo(kr[u][j]), x);
                    x = __builtin_fmaf(q[r][2 * j + 1], T::hi(kr[u][j]), x);
                }
#pragma unroll
                for (int w = 1; w < LPK; w *= 2) x += __shfl_xor(x, w);
                s[u][r] = x;
            }
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mn = m[r];
#pragma unroll
            for (int u = 0; u < kDeep; u++)
                if (ok[u]) mn = fmaxf(mn, s[u][r]);
            const float alpha = __builtin_amdgcn_exp2f((m[r] - mn) * a.c), mc = mn * a.c;
            m[r] = mn;
            l[r] *= alpha;
#pragma unroll
            for (int j = 0; j < 8; j++) o[r][j] *= alpha;
#pragma unroll
            for (int u = 0; u < kDeep; u++) {
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], a.c, -mc));
                if (!ok[u]) p = 0.0f;
                l[r] += p;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    o[r][2 * j] = __builtin_fmaf(p, T::lo(vr[u][j]), o[r][2 * j]);
                    o[r][2 * j + 1] = __builtin_fmaf(p, T::hi(vr[u][j]), o[r][2 * j + 1]);
                }
            }
        }
    }

    // the groups of a wave, then the waves: each weighs by exp2 of its maximum
    __shared__ float so[kWaves][R][8 * LPK], sm[kWaves][R], sl[kWaves][R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        float mn = l[r] > 0.0f || l[r] != l[r] ? m[r] : a.lowest;
#pragma unroll
        for (int w = LPK; w < 64; w *= 2) mn = fmaxf(mn, __shfl_xor(mn, w));
        const float f = l[r] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((m[r] - mn) * a.c);
        l[r] *= f;
#pragma unroll
        for (int w = LPK; w < 64; w *= 2) l[r] += __shfl_xor(l[r], w);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            o[r][j] *= f;
#pragma unroll
            for (int w = LPK; w < 64; w *= 2) o[r][j] += __shfl_xor(o[r][j], w);
        }
        if (lane < LPK) {
#pragma unroll
            for (int j = 0; j < 8; j++) so[wave][r][d + j] = o[r][j];
            if (lane == 0) {
                sm[wave][r] = mn;
                sl[wave][r] = l[r];
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * 8 * LPK; i += kThreads) {
        const int r = i / (8 * LPK), e = i % (8 * LPK);
        if (e >= a.D) continue;
        float mn = a.lowest, sum = 0.0f, x = 0.0f;
        for (int w = 0; w < kWaves; w++)
            if (sl[w][r] != 0.0f) mn = fmaxf(mn, sm[w][r]);
        for (int w = 0; w < kWaves; w++)
            if (sl[w][r] != 0.0f) {
                const float f = __builtin_amdgcn_exp2f((sm[w][r] - mn) * a.c);
                sum = __builtin_fmaf(f, sl[w][r], sum);
                x = __builtin_fmaf(f, so[w][r][e], x);
            }
        const int h = kvh * a.group + r / a.Lq, row = r % a.Lq;
        const int64_t srow = ((int64_t)b * a.H + h) * a.Lq + row;
        const int64_t at = (((int64_t)b * a.Lq + row) * a.H + h) * a.D + e;
        const float y = sum == 0.0f ? 0.0f : x / sum;
        const float stat = sum == 0.0f ? INFINITY : mn * a.c + __builtin_amdgcn_logf(sum);
        if (a.part) {
            a.part[(int64_t)split * a.B * a.Lq * a.H * a.D + at] = y;
            if (e == 0) a.plse[(int64_t)split * a.B * a.H * a.Lq + srow] = stat;
        } else {
            const unsigned v = T::pack(y, 0.0f);
            a.out[at] = (uint16_t)v;
            if (a.rest) a.rest[at] = (uint16_t)T::pack(y - T::lo(v), 0.0f);
            if (a.lse && e == 0) a.lse[srow] = stat;
        }
    }
}

// Joins the ranges of keys: each range's result weighs by its share of the
// row's sum; a range without keys (statistic +inf) takes no part. 2^log threads
// own a row, each V of its channels at a time: rows by shifts and two 32-bit
// divisions. 2 ranges of 16 heads x 1024 rows of 128: 9.5 us, 2.2 TB/s (22 us
// for twice that many rows by a thread and three 64-bit divisions per value).
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(FwdArgs a, int log) {
    // below 2^31: more rows than that fill the chip without ranges
    const unsigned at = blockIdx.x * (kThreads >> log) + (threadIdx.x >> log);
    const unsigned rows = (unsigned)a.B * a.Lq * a.H;
    if (at >= rows) return;
    const unsigned token = at / a.H, h = at % a.H;
    const unsigned b = token / a.Lq, row = token % a.Lq;
    const int64_t srow = ((int64_t)b * a.H + h) * a.Lq + row;
    float mx = -INFINITY;
    bool any = false;
#pragma unroll 8
    for (int s = 0; s < a.splits; s++) {
        const float v = a.plse[(int64_t)s * rows + srow];
        if (v != INFINITY) {
            any = true;
            mx = fmaxf(mx, v);
        }
    }
    const int first = V * (threadIdx.x & ((1 << log) - 1));
    for (int e = first; e < a.D; e += V << log) {
        const int64_t i = (int64_t)at * a.D + e;
        float sum = 0.0f, x[V] = {};
#pragma unroll 4
        for (int s = 0; s < a.splits; s++) {
            const float v = a.plse[(int64_t)s * rows + srow];
            const float* o = a.part + (int64_t)s * rows * a.D + i;
            const float w = v != INFINITY ? __builtin_amdgcn_exp2f(v - mx) : 0.0f;
            sum += w;
            float ov[V];
            if constexpr (V == 4) {
                const f4 q = *reinterpret_cast<const f4*>(o);
#pragma unroll
                for (int j = 0; j < 4; j++) ov[j] = q[j];
            } else {
                ov[0] = *o;
            }
#pragma unroll
            for (int j = 0; j < V; j++) x[j] = __builtin_fmaf(w, ov[j], x[j]);
        }
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = any ? x[j] / sum : 0.0f;
        if constexpr (V == 4) {
            const u2 v = {T::pack(x[0], x[1]), T::pack(x[2], x[3])};
            *reinterpret_cast<u2*>(a.out + i) = v;
            if (a.rest)
                *reinterpret_cast<u2*>(a.rest + i) =
                    u2{T::pack(x[0] - T::lo(v[0]), x[1] - T::hi(v[0])),
                       T::pack(x[2] - T::lo(v[1]), x[3] - T::hi(v[1]))};
        } else {
            const unsigned v = T::pack(x[0], 0.0f);
            a.out[i] = (uint16_t)v;
            if (a.rest) a.rest[i] = (uint16_t)T::pack(x[0] - T::lo(v), 0.0f);
        }
        if (a.lse && e == 0) a.lse[srow] = any ? mx + __builtin_amdgcn_logf(sum) : INFINITY;
    }
}

template <typename T, int V>
void launch_join(const FwdArgs& f, hipStream_t s) {
    int log = 0;
    while (log < 6 && (V << log) < f.D) log++;
    const int64_t rows = (int64_t)f.B * f.Lq * f.H, per = kThreads >> log;
    launch(attention_join_kernel<T, V>, dim3((unsigned)((rows + per - 1) / per)),
           dim3(kThreads), s, f, log);
}

template <typename T>
void launch_main(const FwdArgs& f, hipStream_t s) {
    const dim3 grid((unsigned)f.n), block(kThreads);
    const int dk = (f.D + 15) / 16;
    if (f.pair) {
        launch(attention_pair_kernel<T, 8, 4>, grid, dim3(kPairThreads), s, f);
        return;
    }
    if (dk <= 2) launch(attention_kernel<T, 2, 1>, grid, block, s, f);
    else if (dk <= 3) launch(attention_kernel<T, 3, 2>, grid, block, s, f);
    else if (dk <= 4) launch(attention_kernel<T, 4, 2>, grid, block, s, f);
    else if (dk <= 5) launch(attention_kernel<T, 5, 3>, grid, block, s, f);
    else if (dk <= 6) launch(attention_kernel<T, 6, 3>, grid, block, s, f);
    else if (dk <= 8) launch(attention_kernel<T, 8, 4>, grid, block, s, f);
    else if (dk <= 10) launch(attention_kernel<T, 10, 5>, grid, block, s, f);
    else launch(attention_kernel<T, 16, 8>, grid, block, s, f);
}

template <typename T, int LPK>
void launch_few_rows(const FwdArgs& f, int rows, dim3 grid, hipStream_t s) {
    const dim3 block(kThreads);
    if (rows <= 1) launch(attention_few_kernel<T, LPK, 1>, grid, block, s, f);
    else if (rows <= 2) launch(attention_few_kernel<T, LPK, 2>, grid, block, s, f);
    else if (rows <= 4) launch(attention_few_kernel<T, LPK, 4>, grid, block, s, f);
    else launch(attention_few_kernel<T, LPK, 8>, grid, block, s, f);
}

template <typename T>
void launch_few(const FwdArgs& f, hipStream_t s) {
    const int rows = f.group * f.Lq;
    const dim3 grid((unsigned)(f.B * (f.H / f.group) * f.splits));
    if (f.D <= 32) launch_few_rows<T, 4>(f, rows, grid, s);
    else if (f.D <= 64) launch_few_rows<T, 8>(f, rows, grid, s);
    else if (f.D <= 128) launch_few_rows<T, 16>(f, rows, grid, s);
    else launch_few_rows<T, 32>(f, rows, grid, s);
}

template <typename T>
hipError_t launch_all(const FwdArgs& f, bool few, hipStream_t s) {
    if (few) launch_few<T>(f, s);
    else launch_main<T>(f, s);
    if (f.part) {
        if (f.D % 4 == 0) launch_join<T, 4>(f, s);
        else launch_join<T, 1>(f, s);
    }
    return hipGetLastError();
}

}  // namespace

AttentionPlan attention_plan(const Attention& a, int cus) {
    AttentionPlan p{};
    p.splits = 1;
    const int64_t rows = (int64_t)(a.H / a.KV) * a.Lq;
    // Few rows of a key head, from one or two queries: their own form, which is
    // bound by K and V alone (16 sequences, 1500 keys of 64, us, few | tiles: 1
    // query of 16 heads 25 | 28, of 64 heads in groups of 4 30 | 65, of 8 45 |
    // 64; 2 queries 27.4 | 27.8; 4 queries 30 | 27, 8 queries 59 | 28). Keys that
    // a workgroup holds: 8 x 8 heads of 40, 4096 rows, 77 keys 17.5 | 21.6 over
    // tiles, 128 keys 20 | 27.
    p.form = rows <= 8 && a.Lq <= 2 ? kFew
             : a.Lk >= 1 && a.Lk <= kShortKeys && a.D <= kShortChannels ? kShort
                                                                       : kLong;
    if (p.form == kShort) {
        // blocks of 32 rows for each of a workgroup's four waves: as many as put
        // all workgroups on the chip at once
        const int64_t blocks = (int64_t)a.B * a.H * ((a.Lq + kRows - 1) / kRows);
        const int64_t room = (int64_t)short_waves(a.D) * cus;
        p.per = (int)std::max<int64_t>(1, std::min<int64_t>(8, (blocks + room - 1) / room));
        return p;
    }
    // Two groups of waves where half of the CUs or more get a workgroup and its
    // 256 rows are hardly more than the two or so of 128 that hold them (16 heads
    // of 128, 1024 keys, us: 4096 rows 46 against 51, 2048 rows 40 against 67 in
    // two ranges of keys; 512 sequences' heads with 40 rows each: 29 against 18).
    // Up to 96 channels one group's kernel has four waves a SIMD instead (2 x 64
    // heads x 1024 rows of 64: 62 against 55).
    const int64_t blocks = (a.Lq + kRows - 1) / kRows, pairs = (a.Lq + kPairRows - 1) / kPairRows;
    p.pair = p.form == kLong && a.D > 96 && a.D <= 128 && a.Lk >= 2 * kKeyTile &&
             16 * pairs <= 9 * blocks && 2 * a.B * a.H * pairs >= cus;
    const bool few = p.form == kFew;
    const int64_t unit = few ? 1 : kKeyTile;
    const int64_t units = (a.Lk + unit - 1) / unit;
    const int64_t wgs = few ? (int64_t)a.B * a.KV
                            : (int64_t)a.B * a.H * ((a.Lq + kRows - 1) / kRows);
    const int64_t least = few ? 128 : 2;  // keys or tiles worth a workgroup
    // Ranges of keys until every CU has a workgroup: the join's float32 parts cost
    // more than a second one gains (16 heads x 2048 rows of 64, 1024 keys, us: one
    // per CU 26, two 33), but for few rows, whose parts are small (256 heads' 8
    // rows, 1500 keys: 33 | 28).
    const int64_t room = (few ? 4 : 2 * a.Lq <= kRows ? 2 : 1) * cus;
    int64_t n = std::max<int64_t>(
        1, std::min(room / std::max<int64_t>(wgs, 1), units / least));
    if (p.pair) n = 1;
    n = std::min<int64_t>(n, 64);
    p.per = (int)std::max<int64_t>(1, (units + n - 1) / n);
    p.splits = (int)std::max<int64_t>(1, (units + p.per - 1) / p.per);
    if (p.splits > 1) {
        const int64_t r = (int64_t)a.B * a.H * a.Lq;
        p.ws_bytes = 4 * p.splits * r * (a.D + 1);
    }
    return p;
}

hipError_t launch_attention(const Attention& a, const AttentionPlan& plan, uint16_t* out,
                            uint16_t* rest, float* lse, void* ws, hipStream_t s) {
    if (plan.form == kShort) return launch_attention_short(a, plan.per, out, rest, lse, s);
    FwdArgs f{};
    f.q = a.q;
    f.k = a.k;
    f.v = a.v;
    f.mask = a.mask;
    f.out = out;
    f.rest = rest;
    f.lse = lse;
    f.mask_stride = a.mask_stride;
    std::copy(a.qs, a.qs + 3, f.qs);
    std::copy(a.ks, a.ks + 3, f.ks);
    std::copy(a.vs, a.vs + 3, f.vs);
    f.B = a.B;
    f.Bk = a.Bk;
    f.Lq = a.Lq;
    f.Lk = a.Lk;
    f.H = a.H;
    f.group = a.H / a.KV;
    f.D = a.D;
    f.pair = plan.pair;
    f.qblocks = plan.pair ? (a.Lq + kPairRows - 1) / kPairRows : (a.Lq + kRows - 1) / kRows;
    f.splits = plan.splits;
    f.per = plan.per;
    f.n = a.B * a.H * plan.splits * f.qblocks;
    f.qvec = chunked(a.q, a.qs, a.D);
    f.kvec = chunked(a.k, a.ks, a.D) && close_rows(a.ks[1]);
    f.vvec = chunked(a.v, a.vs, a.D) && close_rows(a.vs[1]);
    f.c = score_scale(a);
    f.lowest = lowest_score(f.c);
    f.flip = a.scale < 0 ? 0x80008000u : 0u;
    f.live = a.scale != 0 ? ~0u : 0u;
    if (plan.splits > 1) {
        f.part = static_cast<float*>(ws);
        f.plse = f.part + (int64_t)plan.splits * a.B * a.Lq * a.H * a.D;
    }
    return a.bf16 ? launch_all<BF16>(f, plan.form == kFew, s)
                  : launch_all<F16>(f, plan.form == kFew, s);
}

}  // namespace nova
