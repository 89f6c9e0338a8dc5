// Attention to up to 128 keys (a prompt's states): a workgroup holds all of them
// in LDS, so a wave's 32 rows take one softmax over registers, without a running
// maximum and without a barrier. The layouts are attention_fwd.hip's: a row per
// lane, S^T = K Q^T, O^T = V^T P^T.
//
// What bounds it: reading the queries and writing the outputs, and for few
// workgroups the chain from the first load to the last store. The next rows are
// on their way while a wave works on its own. 64 heads of 40, 4096 rows, 77 keys:
// 19 us, 2.2 TB/s (20 us the same heads with 128 keys); 160 heads of 64, 1024
// rows: 18 us, 2.3 TB/s; 16 heads of 40, 4096 rows: 8.1 us, 1.3 TB/s.
#include "attention.h"

namespace nova {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

struct ShortArgs {
    const uint16_t *q, *k, *v;
    const uint8_t* mask;
    uint16_t *out, *rest;
    float* lse;
    int64_t qs[3], ks[3], vs[3], mask_stride;
    int B, Bk, Lq, Lk, H, group, D;
    int blocks, per, n;  // workgroups of a head; blocks of 32 rows for each wave; workgroups
    int qvec, kvec, vvec;
    float c, lowest;  // lowest: see lowest_score
    unsigned flip, live;
};

// NB: blocks of 32 keys.
template <typename T, int DK, int NB>
__global__ __launch_bounds__(kThreads, short_waves(16 * DK)) void attention_short_kernel(ShortArgs a) {
    constexpr int DV = (DK + 1) / 2, kStride = 16 * DK + 8;
    typedef Padded<kStride> L;
    // the last rows' reads of channels past D stay inside
    __shared__ __attribute__((aligned(16))) uint16_t kt[32 * NB * kStride];
    __shared__ __attribute__((aligned(16))) uint16_t vt[32 * NB * kStride + 64];
    __shared__ __attribute__((aligned(16))) float bias[32 * NB];

    const int id = xcd_remap(blockIdx.x, a.n);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block = id % a.blocks, bh = id / a.blocks;
    const int h = bh % a.H, b = bh / a.H;
    const int kvh = h / a.group, bk = a.Bk == 1 ? 0 : b;
    const uint16_t* qp = a.q + b * a.qs[0] + h * a.qs[2];
    const int row0 = (block * kWaves + wave) * a.per * 32;

    u4 qf[DK];
    auto load_q = [&](int row, u4(&f)[DK]) {
        load_row<DK>(qp + min(row, a.Lq - 1) * a.qs[1], row < a.Lq, half, a.D, a.qvec, f);
    };
    load_q(row0 + (lane & 31), qf);

    unsigned keep[NB];
    kept_keys<NB>(a.mask ? a.mask + b * a.mask_stride : nullptr, a.Lk, keep, bias);
    {
        const uint16_t* kp = a.k + bk * a.ks[0] + kvh * a.ks[2];
        const uint16_t* vp = a.v + bk * a.vs[0] + kvh * a.vs[2];
        fill_keys<DK, NB>(kt, vt, kp, vp, a.ks[1], a.vs[1], keep, a.Lk, a.D, a.kvec && a.vvec,
                          tid, kThreads);
    }
    __syncthreads();

    for (int i = 0; i < a.per; i++) {
        const int row = row0 + 32 * i + (lane & 31);
        if (row0 + 32 * i >= a.Lq) break;
#pragma unroll
        for (int s = 0; s < DK; s++) qf[s] = (qf[s] & a.live) ^ a.flip;
        f16v s[NB];
        float m = a.lowest;
#pragma unroll
        for (int kb = 0; kb < NB; kb++) {
            s[kb] = start_scores(bias + 32 * kb, half);
#pragma unroll
            for (int st = 0; st < DK; st++)
                s[kb] = T::mfma(L::rows(kt, lane, 32 * kb, st), qf[st], s[kb]);
        }
        if (i + 1 < a.per) load_q(row + 32, qf);
#pragma unroll
        for (int kb = 0; kb < NB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) m = fmaxf(m, s[kb][r]);
        m = max_halves(m);
        const float mc = m * a.c;
        float l = 0.0f;
        f16v o[DV];
#pragma unroll
        for (int d = 0; d < DV; d++) o[d] = f16v{};
#pragma unroll
        for (int kb = 0; kb < NB; kb++) {
            unsigned p[8];
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], a.c, -mc));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], a.c, -mc));
                l += x + y;
                p[r / 2] = T::pack(x, y);
            }
#pragma unroll
            for (int d = 0; d < DV; d++)
#pragma unroll
                for (int g = 0; g < 2; g++)
                    o[d] = T::mfma(L::turned(vt, lane, 32 * kb + 16 * g, d),
                                   u4{p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]}, o[d]);
        }
        l = add_halves(l);
        if (row >= a.Lq) continue;
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays
        if (a.lse && half == 0)
            a.lse[((int64_t)b * a.H + h) * a.Lq + row] =
                l == 0.0f ? INFINITY : mc + __builtin_amdgcn_logf(l);
        uint16_t* p = a.out + (((int64_t)b * a.Lq + row) * a.H + h) * a.D;
        store_row<T, DV>(p, a.rest ? a.rest + (p - a.out) : nullptr, o, inv, half, a.D);
    }
}

template <typename T, int DK>
void launch_keys(const ShortArgs& f, hipStream_t s) {
    const dim3 grid((unsigned)f.n), block(kThreads);
    if (f.Lk <= 64) launch(attention_short_kernel<T, DK, 2>, grid, block, s, f);
    else if (f.Lk <= 96) launch(attention_short_kernel<T, DK, 3>, grid, block, s, f);
    else launch(attention_short_kernel<T, DK, 4>, grid, block, s, f);
}

template <typename T>
hipError_t launch_all(const ShortArgs& f, hipStream_t s) {
    const int dk = (f.D + 15) / 16;
    if (dk <= 3) launch_keys<T, 3>(f, s);
    else if (dk <= 4) launch_keys<T, 4>(f, s);
    else if (dk <= 5) launch_keys<T, 5>(f, s);
    else if (dk <= 8) launch_keys<T, 8>(f, s);
    else launch_keys<T, 10>(f, s);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_short(const Attention& a, int per, uint16_t* out, uint16_t* rest,
                                  float* lse, hipStream_t s) {
    ShortArgs f{};
    f.q = a.q;
    f.k = a.k;
    f.v = a.v;
    f.mask = a.mask;
    f.out = out;
    f.rest = rest;
    f.lse = lse;
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
    f.group = a.H / a.KV;
    f.D = a.D;
    f.per = per;
    f.blocks = (a.Lq + 32 * kWaves * per - 1) / (32 * kWaves * per);
    f.n = a.B * a.H * f.blocks;
    f.qvec = chunked(a.q, a.qs, a.D);
    f.kvec = chunked(a.k, a.ks, a.D);
    f.vvec = chunked(a.v, a.vs, a.D);
    f.c = score_scale(a);
    f.lowest = lowest_score(f.c);
    f.flip = a.scale < 0 ? 0x80008000u : 0u;
    f.live = a.scale != 0 ? ~0u : 0u;
    return a.bf16 ? launch_all<BF16>(f, s) : launch_all<F16>(f, s);
}

}  // namespace nova
