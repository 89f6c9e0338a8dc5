// Gradients of attention to up to 128 keys (see attention_bwd.hip for the
// formulas), in one kernel: a workgroup of NB waves holds K and V in LDS, walks
// its range of the query tiles (32 NB rows: every head and row that reads these
// keys) and works on each in two turns.
//
//   a wave owns 32 query rows, one per lane, against all keys: S^T, dP^T, P, ds,
//   delta from its own registers (exact: the forward's output is not read), dq;
//   P, then ds, goes to LDS as rows;
//
//   then a wave owns 32 keys, one per lane, against all the tile's rows: dv and
//   dk, accumulated over the whole range, from P or ds and dO or Q, all read
//   transposed.
//
// P and ds are computed once for all three gradients. What bounds it: neither
// bytes nor the matrix unit, but the chain of the two turns in the one or two
// workgroups that a CU's LDS holds. 64 heads of 40, 4096 rows, 77 keys: 50 us and
// 4 us for the join of the workgroups' sums (dq, dk and dv over tiles: 80 us).
//
// float16: P enters times 2^10, ds times a power of two: in dq one of the row's
// own, in dk, whose sums run over the rows, one that the workgroup shares. That
// one moves, with the sums so far, only when a tile's largest value would leave
// the type's range: a dk's terms are off by up to 2^-32 of the largest ds that
// the workgroup has met. (With the shared one in dq too, rows whose gradients
// were 2^-20 of others' had errors of 1.6e-3, the type's own being 3e-4.)
#include "attention.h"

namespace nova {

namespace {

struct ShortBwdArgs {
    const uint16_t *q, *k, *v, *go;
    const uint8_t* mask;
    const float* lse;
    uint16_t *dq, *dk, *dv;
    float* part;
    int64_t qs[3], ks[3], vs[3], mask_stride;
    int B, Bk, Lq, Lk, H, KV, group, D;
    int tiles;  // of a head's rows
    int units, splits, per, n;
    int qvec, kvec, vvec, ovec;
    float c, scale;
    unsigned flip, live;
};

// Waves per SIMD that the registers are cut for: two where nothing spills.
constexpr int short_bwd_waves(int DK, int NB) { return NB <= 3 && DK <= 4 ? 2 : 1; }

template <typename T, int DK, int NB>
__global__ __launch_bounds__(64 * NB, short_bwd_waves(DK, NB)) void attention_short_bwd_kernel(
    ShortBwdArgs a) {
    constexpr int DV = (DK + 1) / 2, kStride = 16 * DK + 8, kThreads = 64 * NB, kRows = 32 * NB;
    constexpr int kPStride = 32 * NB + 8;
    typedef Padded<kStride> L;
    typedef Padded<kPStride> LP;
    // reads of channels past D in a tile's last rows stay inside
    constexpr int kTile = kRows * kStride + 64;
    __shared__ __attribute__((aligned(16))) uint16_t lds[4 * kTile + kRows * kPStride];
    __shared__ __attribute__((aligned(16))) float bias[kRows];
    __shared__ float tops[NB];
    static_assert(sizeof(lds) + sizeof(bias) + sizeof(tops) <= 160 * 1024, "LDS of a CU");
    uint16_t *kt = lds, *vt = kt + kTile, *qt = vt + kTile, *gt = qt + kTile, *pt = gt + kTile;

    const int id = xcd_remap(blockIdx.x, a.n);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = id % a.splits;
    const int kvh = id / a.splits % a.KV, bk = id / a.splits / a.KV;

    unsigned keep[NB];
    kept_keys<NB>(a.mask ? a.mask + bk * a.mask_stride : nullptr, a.Lk, keep, bias);
    {
        const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
        const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
        fill_keys<DK, NB>(kt, vt, kp, vp, a.ks[1], a.vs[1], keep, a.Lk, a.D, a.kvec && a.vvec,
                          tid, kThreads);
    }

    f16v dk[DV], dv[DV];
#pragma unroll
    for (int d = 0; d < DV; d++) dk[d] = dv[d] = f16v{};
    float f = T::kHalf ? 0.0f : 1.0f;  // ds enters products times f; 0: none seen yet

    const int u0 = split * a.per, u1 = min(a.units, u0 + a.per);
    const int mine = wave * 32 + (lane & 31);
    // place of a row's quad of keys in the P tile
    uint16_t* prow = pt + mine * kPStride + 4 * half;

    u4 qf[DK], gf[DK];
    float lse;
    auto fetch = [&](const QueryTile& p) {
        const int row = p.tile * kRows + mine, h = kvh * a.group + p.head, b = p.seq;
        const bool live = row < a.Lq;
        const int at = min(row, a.Lq - 1);
        const int64_t orow = (((int64_t)b * a.Lq + at) * a.H + h) * a.D;
        load_row<DK>(a.q + b * a.qs[0] + h * a.qs[2] + at * a.qs[1], live, half, a.D, a.qvec, qf);
        load_row<DK>(a.go + orow, live, half, a.D, a.ovec, gf);
        lse = a.lse[((int64_t)b * a.H + h) * a.Lq + at];
        if (!live) lse = INFINITY;
    };
    QueryTile now(u0, a.tiles, a.group, a.Bk == 1 ? 0 : bk), after = now;
    if (u0 < u1) fetch(now);
    for (int u = u0; u < u1; u++) {
        lds_barrier();  // the last tile's reads are over (and K and V are there)
#pragma unroll
        for (int s = 0; s < DK; s++) {
            qf[s] = (qf[s] & a.live) ^ a.flip;
            *reinterpret_cast<u4*>(qt + mine * kStride + 16 * s + 8 * half) = qf[s];
            *reinterpret_cast<u4*>(gt + mine * kStride + 16 * s + 8 * half) = gf[s];
        }
        f16v s[NB], g[NB];
#pragma unroll
        for (int kb = 0; kb < NB; kb++) {
            s[kb] = start_scores(bias + 32 * kb, half);
            g[kb] = f16v{};
#pragma unroll
            for (int st = 0; st < DK; st++) {
                s[kb] = T::mfma(L::rows(kt, lane, 32 * kb, st), qf[st], s[kb]);
                g[kb] = T::mfma(L::rows(vt, lane, 32 * kb, st), gf[st], g[kb]);
            }
        }
        constexpr float kUp = T::kHalf ? 10.0f : 0.0f;
        const float shift = kUp - lse;
        float delta = 0.0f;
#pragma unroll
        for (int kb = 0; kb < NB; kb++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.c, shift));
                delta = __builtin_fmaf(s[kb][r], g[kb][r], delta);
            }
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<u2*>(prow + 32 * kb + acc_row(r)) =
                    u2{T::pack(s[kb][r], s[kb][r + 1]), T::pack(s[kb][r + 2], s[kb][r + 3])};
        }
        delta = add_halves(delta) * (T::kHalf ? 0x1p-10f : 1.0f);
        float top = 0.0f;
#pragma unroll
        for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[kb][r] *= g[kb][r] - delta;
                if (T::kHalf) top = fmaxf(top, fabsf(s[kb][r]));
            }
        int up = 0;  // ds enters the row's own product, dq, times 2^up
        if (T::kHalf) {
            up = half_range(max_halves(top));
            top = max_wave(top);
            if (lane == 0) tops[wave] = top;
        }
        lds_barrier();  // Q, dO, P and the waves' tops are there

        // dv of this wave's keys
#pragma unroll
        for (int x = 0; x < 2 * NB; x++) {
            const u4 p = LP::turned(pt, lane, 16 * x, wave);
#pragma unroll
            for (int d = 0; d < DV; d++)
                dv[d] = T::mfma(L::turned(gt, lane, 16 * x, d), p, dv[d]);
        }
        if (T::kHalf) {
            top = 0.0f;
#pragma unroll
            for (int w = 0; w < NB; w++) top = fmaxf(top, tops[w]);
            top = __builtin_bit_cast(
                float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, top)));
            if (top * f > 32768.0f || (f == 0.0f && top > 0.0f)) {
                const float to = __builtin_ldexpf(1.0f, half_range(top));
                const float fix = f == 0.0f ? 1.0f : to / f;
                f = to;
#pragma unroll
                for (int d = 0; d < DV; d++) dk[d] *= fix;
            }
        }
        unsigned ds[NB][8];
        const float fq = __builtin_ldexpf(1.0f, up);
#pragma unroll
        for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r += 2)
                ds[kb][r / 2] = T::pack(s[kb][r] * fq, s[kb][r + 1] * fq);
        lds_barrier();  // P is read
        // from the row's power of two to the shared one: at most 2^8 times
        const float to_all = __builtin_ldexpf(f, -up);
#pragma unroll
        for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<u2*>(prow + 32 * kb + acc_row(r)) =
                    u2{T::scaled(ds[kb][r / 2], to_all), T::scaled(ds[kb][r / 2 + 1], to_all)};
        // dq of this wave's rows
        f16v acc[DV];
#pragma unroll
        for (int d = 0; d < DV; d++) acc[d] = f16v{};
#pragma unroll
        for (int x = 0; x < 2 * NB; x++) {
            const unsigned* pp = &ds[x >> 1][4 * (x & 1)];
#pragma unroll
            for (int d = 0; d < DV; d++)
                acc[d] = T::mfma(L::turned(kt, lane, 16 * x, d),
                                 u4{pp[0], pp[1], pp[2], pp[3]}, acc[d]);
        }
        after.next(a.tiles, a.group);
        if (u + 1 < u1) fetch(after);
        {
            const int row = now.tile * kRows + mine, h = kvh * a.group + now.head, b = now.seq;
            if (row < a.Lq) {
                float of = a.flip ? -a.scale : a.scale;
                if (T::kHalf) of = __builtin_ldexpf(of, -up - 10);
                uint16_t* p = a.dq + (((int64_t)b * a.Lq + row) * a.H + h) * a.D;
                store_row<T, DV>(p, nullptr, acc, of, half, a.D);
            }
        }
        lds_barrier();  // ds is there
        // dk of this wave's keys
#pragma unroll
        for (int x = 0; x < 2 * NB; x++) {
            const u4 p = LP::turned(pt, lane, 16 * x, wave);
#pragma unroll
            for (int d = 0; d < DV; d++)
                dk[d] = T::mfma(L::turned(qt, lane, 16 * x, d), p, dk[d]);
        }
        now = after;
    }

    if (mine >= a.Lk) return;
    // the queries already carry the scale's sign
    float fk = a.scale, fv = 1.0f;
    if (T::kHalf) {
        fk = f == 0.0f ? 0.0f : fk / f * 0x1p-10f;
        fv = 0x1p-10f;
    }
    const int64_t krow = (((int64_t)bk * a.Lk + mine) * a.KV + kvh) * a.D;
    const int64_t all = (int64_t)a.Bk * a.Lk * a.KV * a.D;
#pragma unroll
    for (int d = 0; d < DV; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + acc_row(r) + 4 * half;
            if (a.part) {
                float* to = a.part + 2 * split * all + krow;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (e + j < a.D) {
                        to[e + j] = dk[d][r + j] * fk;
                        to[all + e + j] = dv[d][r + j] * fv;
                    }
            } else {
                store_quad(a.dk + krow, e, a.D,
                           u2{T::pack(dk[d][r] * fk, dk[d][r + 1] * fk),
                              T::pack(dk[d][r + 2] * fk, dk[d][r + 3] * fk)});
                store_quad(a.dv + krow, e, a.D,
                           u2{T::pack(dv[d][r] * fv, dv[d][r + 1] * fv),
                              T::pack(dv[d][r + 2] * fv, dv[d][r + 3] * fv)});
            }
        }
}

template <typename T, int DK>
void launch_keys(const ShortBwdArgs& f, hipStream_t s) {
    const dim3 grid((unsigned)f.n);
    if (f.Lk <= 64) launch(attention_short_bwd_kernel<T, DK, 2>, grid, dim3(128), s, f);
    else if (f.Lk <= 96) launch(attention_short_bwd_kernel<T, DK, 3>, grid, dim3(192), s, f);
    else if constexpr (DK <= kShortDeep)
        launch(attention_short_bwd_kernel<T, DK, 4>, grid, dim3(256), s, f);
}

template <typename T>
hipError_t launch_all(const ShortBwdArgs& f, hipStream_t s) {
    const int dk = (f.D + 15) / 16;
    if (dk <= 3) launch_keys<T, 3>(f, s);
    else if (dk <= 4) launch_keys<T, 4>(f, s);
    else if (dk <= 5) launch_keys<T, 5>(f, s);
    else if (dk <= 8) launch_keys<T, 8>(f, s);
    else launch_keys<T, 10>(f, s);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_short_bwd(const Attention& a, const AttentionBwdPlan& plan,
                                      const float* lse, const uint16_t* go, uint16_t* dq,
                                      uint16_t* dk, uint16_t* dv, float* part, hipStream_t s) {
    ShortBwdArgs f{};
    f.q = a.q;
    f.k = a.k;
    f.v = a.v;
    f.go = go;
    f.mask = a.mask;
    f.lse = lse;
    f.dq = dq;
    f.dk = dk;
    f.dv = dv;
    f.part = part;
    f.mask_stride = a.mask_stride;
    for (int i = 0; i < 3; i++) {
        f.qs[i] = a.qs[i];
        f.ks[i] = a.ks[i];
        f.vs[i] = a.vs[i];
    }
    f.B = a.B;
    f.Bk = a.Bk;
    f.Lq = a.Lq;
    f.Lk = a.Lk;
    f.H = a.H;
    f.KV = a.KV;
    f.group = a.H / a.KV;
    f.D = a.D;
    f.tiles = (a.Lq + plan.rows - 1) / plan.rows;
    f.units = plan.units;
    f.splits = plan.splits;
    f.per = plan.per;
    f.n = a.Bk * a.KV * plan.splits;
    const int64_t os[3] = {a.D, a.D, a.D};
    f.qvec = chunked(a.q, a.qs, a.D);
    f.kvec = chunked(a.k, a.ks, a.D);
    f.vvec = chunked(a.v, a.vs, a.D);
    f.ovec = chunked(go, os, a.D);
    f.scale = a.scale < 0 ? -a.scale : a.scale;
    f.c = score_scale(a);
    f.flip = a.scale < 0 ? 0x80008000u : 0u;
    f.live = a.scale != 0 ? ~0u : 0u;
    return a.bf16 ? launch_all<BF16>(f, s) : launch_all<F16>(f, s);
}

}  // namespace nova
