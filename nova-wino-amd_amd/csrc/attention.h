// Device code shared by the attention kernels (attention_fwd.hip,
// attention_bwd.hip): element types, operand layouts, tile staging.
#pragma once

#include "nova_internal.h"
#include "nova_tile_math.h"

namespace nova {

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct F16 {
    static constexpr bool kHalf = true;
    static __device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                      __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    // two values, each rounded to nearest even
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{x, y}, h2));
    }
    // two packed values times a power of two
    static __device__ __forceinline__ unsigned scaled(unsigned v, float f) {
        const _Float16 x = (_Float16)f;
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(h2, v) * h2{x, x});
    }
    static __device__ __forceinline__ float lo(unsigned v) {
        return (float)__builtin_bit_cast(h2, v)[0];
    }
    static __device__ __forceinline__ float hi(unsigned v) {
        return (float)__builtin_bit_cast(h2, v)[1];
    }
};

struct BF16 {
    static constexpr bool kHalf = false;
    static __device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a),
                                                       __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{x, y}, b2));
    }
    static __device__ __forceinline__ unsigned scaled(unsigned v, float) { return v; }  // by 1
    static __device__ __forceinline__ float lo(unsigned v) {
        return __builtin_bit_cast(float, v << 16);
    }
    static __device__ __forceinline__ float hi(unsigned v) {
        return __builtin_bit_cast(float, v & 0xffff0000u);
    }
};

// Keys per tile of the kernels that walk the keys, and tiles whose masks one
// fill of the bitmap in LDS holds.
constexpr int kKeyTile = 64;
constexpr int kMaskTiles = 128;

// Row of accumulator r of a 32x32 product in lane l is acc_row(r) + 4 * (l / 32).
constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

// 8 elements of a row from channel d on, zeros from channel D on. vec: rows
// start on 16 bytes and D is a multiple of 8, so a chunk is one load.
__device__ __forceinline__ u4 load_chunk(const uint16_t* row, int d, int D, int vec) {
    u4 r = {0, 0, 0, 0};
    if (d < D) {
        if (vec) {
            r = *reinterpret_cast<const u4*>(row + d);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                unsigned w = 0;
                if (d + 2 * j < D) w = row[d + 2 * j];
                if (d + 2 * j + 1 < D) w |= (unsigned)row[d + 2 * j + 1] << 16;
                r[j] = w;
            }
        }
    }
    return r;
}

// The chunks of a row that lane half `half` holds of a 32x32x16 product's B
// operand, zeros past D and where the row is not live (row may then be any
// readable one). One branch around the loads; with vec they are unconditional.
template <int DK>
__device__ __forceinline__ void load_row(const uint16_t* row, bool live, int half, int D, int vec,
                                         u4 (&f)[DK]) {
    asm volatile("" : "+s"(D));  // as in store_row
    if (vec) {
#pragma unroll
        for (int s = 0; s < DK; s++)
            f[s] = *reinterpret_cast<const u4*>(row + min(16 * s + 8 * half, D - 8));
#pragma unroll
        for (int s = 0; s < DK; s++) {
            const unsigned on = live && 16 * s + 8 * half < D ? ~0u : 0u;
            f[s] &= on;
        }
    } else {
        for (int s = 0; s < DK; s++) {
            u4 x = {0, 0, 0, 0};
            if (live) x = load_chunk(row, 16 * s + 8 * half, D, 0);
#pragma unroll
            for (int i = 0; i < DK; i++) f[i] = i == s ? x : f[i];
        }
    }
}

// Rows of LDS, STRIDE elements apart (8 more than a multiple of 16, so that a
// product's operand reads spread over the banks): operands of 32x32x16
// products. The orders are Tile's.
template <int STRIDE>
struct Padded {
    // Rows r0 .. r0 + 31, columns 16 * st on, contracted over columns.
    static __device__ __forceinline__ u4 rows(const uint16_t* t, int lane, int r0, int st) {
        return *reinterpret_cast<const u4*>(t + (r0 + (lane & 31)) * STRIDE + 16 * st +
                                            8 * (lane >> 5));
    }
    // Columns 32 * d on, contracted over rows r0 .. r0 + 15.
    static __device__ __forceinline__ u4 turned(const uint16_t* t, int lane, int r0, int d) {
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const int row = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
        const int col = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const uint16_t* p = t + row * STRIDE + col;
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p));
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * STRIDE));
        const u2 a = __builtin_bit_cast(u2, x), b = __builtin_bit_cast(u2, y);
        return u4{a[0], a[1], b[0], b[1]};
    }
};

// Keys up to which a workgroup holds all of them (attention_short_*.hip), and
// the channels (in 16s) up to which its backward holds more than 96 keys: K, V,
// Q, dO and P of a tile have to fit the LDS of a CU.
constexpr int kShortKeys = 128;
constexpr int kShortChannels = 160;
constexpr int kShortDeep = 5;

// Workgroups of the short forward that a CU holds (waves per SIMD).
constexpr int short_waves(int D) { return D <= 64 ? 3 : D <= 128 ? 2 : 1; }

// Kept keys as bits, the same in all waves, and the scores' start: 0, or -inf
// for a key that takes no part (bias: LDS, 32 * NB floats).
template <int NB>
__device__ __forceinline__ void kept_keys(const uint8_t* mask, int Lk, unsigned (&keep)[NB],
                                          float* bias) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < NB; i += 2) {
        const int j = 32 * i + lane;
        bool in = j < Lk;
        if (mask && in) in = mask[j] != 0;
        const uint64_t v = __ballot(in);
        keep[i] = (unsigned)v;
        if (i + 1 < NB) keep[i + 1] = (unsigned)(v >> 32);
        if ((int)threadIdx.x < 64 && j < 32 * NB) bias[j] = in ? 0.0f : -INFINITY;
    }
}

// A block's scores before its products: bias of its keys.
__device__ __forceinline__ f16v start_scores(const float* bias, int half) {
    f16v s;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const f4 b = *reinterpret_cast<const f4*>(bias + acc_row(r) + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; e++) s[r + e] = b[e];
    }
    return s;
}

// K and V of all keys, 32 * NB rows of 16 * DK + 8 elements, zeros for keys that
// are not kept and past D. Lk: at least 1.
template <int DK, int NB>
__device__ __forceinline__ void fill_keys(uint16_t* kt, uint16_t* vt, const uint16_t* kp,
                                          const uint16_t* vp, int64_t ks, int64_t vs,
                                          const unsigned (&keep)[NB], int Lk, int D, int vec,
                                          int tid, int threads) {
    constexpr int kChunks = 2 * DK, kStride = 16 * DK + 8;
    auto at = [&](int s, int* r, int* d, bool* ok) {
        *r = s / kChunks;
        *d = 8 * (s % kChunks);
        unsigned bits = 0;
#pragma unroll
        for (int e = 0; e < NB; e++) bits = (*r >> 5) == e ? keep[e] : bits;
        *ok = ((bits >> (*r & 31)) & 1) && *d < D;
    };
    if (vec) {
#pragma unroll 4
        for (int s = tid; s < 32 * NB * kChunks; s += threads) {
            int r, d;
            bool ok;
            at(s, &r, &d, &ok);
            const int row = min(r, Lk - 1), col = min(d, D - 8);
            u4 x = *reinterpret_cast<const u4*>(kp + row * ks + col);
            u4 y = *reinterpret_cast<const u4*>(vp + row * vs + col);
            if (!ok) x = y = u4{0, 0, 0, 0};
            *reinterpret_cast<u4*>(kt + r * kStride + d) = x;
            *reinterpret_cast<u4*>(vt + r * kStride + d) = y;
        }
    } else {
        for (int s = tid; s < 32 * NB * kChunks; s += threads) {
            int r, d;
            bool ok;
            at(s, &r, &d, &ok);
            u4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (ok) {
                x = load_chunk(kp + r * ks, d, D, 0);
                y = load_chunk(vp + r * vs, d, D, 0);
            }
            *reinterpret_cast<u4*>(kt + r * kStride + d) = x;
            *reinterpret_cast<u4*>(vt + r * kStride + d) = y;
        }
    }
}

// A tile of 64 rows x COLS channels (a multiple of 64) in LDS: 16-byte chunks,
// row by row, the chunks of each group of eight in an order of their own for
// each row (XOR with swizzle(row)), so that 8 rows' chunks of one number, and
// the 4 rows x 32 bytes that 16 lanes of a transposing load read, lie in
// different banks without padding, which direct loads to LDS cannot leave.
__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

// An offset past the end of every resource that a tile is loaded through: the
// load brings zeros.
constexpr int kOutside = 0x7ffffff0;

template <int COLS>
struct Tile {
    static constexpr int kChunks = COLS / 8;
    static constexpr int kElems = 64 * COLS;

    // Lane constants of the operand reads.
    struct Lane {
        int rows[4], turned[2];
        __device__ __forceinline__ explicit Lane(int lane) {
            const int half = lane >> 5;
#pragma unroll
            for (int i = 0; i < 4; i++)
                rows[i] = (lane & 31) * COLS + 8 * ((2 * i + half) ^ swizzle(lane));
            const int row = 4 * half + ((lane & 15) >> 2);
            const int chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
            for (int i = 0; i < 2; i++)
                turned[i] = row * COLS + 8 * ((4 * i + chunk) ^ swizzle(row)) + 4 * (lane & 1);
        }
    };

    // Rows r0 .. r0 + 31 (r0 a multiple of 32), channels 16 * st on, as the A
    // operand of a product that contracts over channels.
    static __device__ __forceinline__ u4 rows(const uint16_t* t, const Lane& l, int r0, int st) {
        return *reinterpret_cast<const u4*>(t + l.rows[st & 3] + r0 * COLS + 64 * (st >> 2));
    }

    // A operand of a 32x32x16 product whose rows are channels 32 * d on and
    // whose contraction runs over 16 of the tile's rows from r0 (a multiple of
    // 16) on, transposed by the load. The contraction slots of lanes 0-31 hold
    // rows {0-3, 8-11} and of lanes 32-63 rows {4-7, 12-15}: the rows that a
    // product's accumulators leave in those lanes, so accumulators go into the
    // next product as its B operand without leaving their lane.
    static __device__ __forceinline__ u4 turned(const uint16_t* t, const Lane& l, int r0, int d) {
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const uint16_t* p = t + l.turned[d & 1] + r0 * COLS + 64 * (d >> 1);
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p));
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * COLS));
        const u2 a = __builtin_bit_cast(u2, x), b = __builtin_bit_cast(u2, y);
        return u4{a[0], a[1], b[0], b[1]};
    }

    // Fills tiles from rows in memory, THREADS threads.
    template <int THREADS>
    struct FillBy {
        static constexpr int kLoads = 64 * kChunks / THREADS;  // chunks of a thread
        int off[kLoads];  // of the chunk that the thread loads, in bytes; kOutside: past D
        __device__ __forceinline__ FillBy(int tid, int64_t stride, int D) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int s = i * THREADS + tid, r = s / kChunks, pos = s % kChunks;
                const int c = (pos & ~7) | ((pos ^ swizzle(r)) & 7);
                off[i] = 8 * c < D ? (int)(2 * (r * stride + 8 * c)) : kOutside;
            }
        }
        // Rows with their bit set in keep; the others become zeros. direct: rows
        // come in whole chunks and 64 of them span less than 2 GB: straight to
        // LDS (counted in vmcnt), else through registers.
        __device__ __forceinline__ void operator()(uint16_t* t, const uint16_t* row0,
                                                   int64_t stride, uint64_t keep, int D,
                                                   int direct, int tid) const {
            if (direct) {
                const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<uint16_t*>(row0), 0, (int)(2 * (63 * stride + D)), 0x00020000);
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    const int r = (i * THREADS + tid) / kChunks;
                    load_lds16(rs, t + (i * THREADS + wave * 64) * 8,
                               (keep >> r) & 1 ? off[i] : kOutside, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kLoads; i++) {
                    const int s = i * THREADS + tid, r = s / kChunks, pos = s % kChunks;
                    const int c = (pos & ~7) | ((pos ^ swizzle(r)) & 7);
                    u4 v = {0, 0, 0, 0};
                    if ((keep >> r) & 1) v = load_chunk(row0 + r * stride, 8 * c, D, 0);
                    *reinterpret_cast<u4*>(t + s * 8) = v;
                }
            }
        }
    };
    typedef FillBy<256> Fill;
};

// Channels at .. at + 3 of a dense row of D, those that exist.
__device__ __forceinline__ void store_quad(uint16_t* row, int at, int D, u2 v) {
    if ((D & 3) == 0) {  // rows then start on 8 bytes
        if (at < D) *reinterpret_cast<u2*>(row + at) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (at + e < D) row[at + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
}

// The accumulators of a row's channels, times f, into the row, and into rest (or
// null) what their rounding dropped.
template <typename T, int DV>
__device__ __forceinline__ void store_row(uint16_t* row, uint16_t* rest, const f16v (&o)[DV],
                                          float f, int half, int D) {
    // the comparisons with D are not worth registers around a caller's loop
    asm volatile("" : "+s"(D));
#pragma unroll
    for (int d = 0; d < DV; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const float x = o[d][r] * f, y = o[d][r + 1] * f;
            const float z = o[d][r + 2] * f, w = o[d][r + 3] * f;
            const int at = 32 * d + acc_row(r) + 4 * half;
            const u2 v = {T::pack(x, y), T::pack(z, w)};
            store_quad(row, at, D, v);
            if (rest)
                store_quad(rest, at, D,
                           u2{T::pack(x - T::lo(v[0]), y - T::hi(v[0])),
                              T::pack(z - T::lo(v[1]), w - T::hi(v[1]))});
        }
}

// x and that of the lane 32 away, combined: swapping halves between two copies
// of x leaves its lower half in both halves of one, its upper half in both of
// the other.
__device__ __forceinline__ float max_halves(float x) {
    const int u = __builtin_bit_cast(int, x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (int)s[0]), __builtin_bit_cast(float, (int)s[1]));
}
__device__ __forceinline__ float add_halves(float x) {
    const int u = __builtin_bit_cast(int, x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (int)s[0]) + __builtin_bit_cast(float, (int)s[1]);
}

// Largest x (x >= 0) of the wave, in a scalar register: lane permutations in the
// instructions themselves, then the four rows' values.
template <int CTRL>
__device__ __forceinline__ float max_dpp(float x) {
    return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                                  0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf,
                                                  true)));
}
__device__ __forceinline__ float max_wave(float x) {
    x = max_dpp<0xB1>(x);   // lane ^ 1
    x = max_dpp<0x4E>(x);   // lane ^ 2
    x = max_dpp<0x141>(x);  // mirrored in 8
    x = max_dpp<0x140>(x);  // mirrored in 16
    const int u = __builtin_bit_cast(int, x);
    const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(u, 0));
    const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(u, 16));
    const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(u, 32));
    const float d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(u, 48));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// x, -100 to 100, such that 2^x brings a float16 product's operands of up to
// `largest` (>= 0) to between 2^7 and 2^8: eight bits of room above, for later
// ones.
__device__ __forceinline__ int half_range(float largest) {
    int e;
    (void)__builtin_frexpf(largest, &e);  // largest < 2^e
    return largest > 0.0f ? min(max(8 - e, -100), 100) : 100;
}

// Place of a unit of the walk over query tiles: every tile of every query head
// that reads a key head, of every sequence that reads the keys.
struct QueryTile {
    int tile, head, seq;  // tile of the head's rows; head of the group; sequence
    __device__ __forceinline__ QueryTile(int u, int tiles, int group, int seq0) {
        const int hb = u / tiles;
        tile = u - hb * tiles;
        const int s = hb / group;
        head = hb - s * group;
        seq = seq0 + s;
    }
    __device__ __forceinline__ void next(int tiles, int group) {
        if (++tile == tiles) {
            tile = 0;
            if (++head == group) {
                head = 0;
                seq++;
            }
        }
    }
};

// The kept keys of a tile of 64 by the bitmap's words, in scalar registers.
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
    return (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)x) |
           (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(x >> 32)) << 32;
}

// Steps through the tiles [t, t1) of 64 keys that keep a key. bits: LDS,
// kMaskTiles words. Every thread of the workgroup calls it alike (a new stretch
// of the mask passes barriers). waves: of the workgroup.
struct KeyTiles {
    int t, t1, w1, Lk, waves;
    const uint8_t* mask;
    uint64_t* bits;
    __device__ __forceinline__ KeyTiles(int first, int end, int keys, const uint8_t* m,
                                        uint64_t* b, int n)
        : t(first - 1), t1(end), w1(first), Lk(keys), waves(n), mask(m), bits(b) {}
    // Number of the next such tile and its kept keys; 0 kept: there is none.
    __device__ __forceinline__ int next(uint64_t* kept) {
        for (t++; t < t1; t++) {
            if (mask == nullptr) {
                const int n = Lk - t * kKeyTile;
                *kept = n >= kKeyTile ? ~0ull : (1ull << n) - 1;
                return t;
            }
            if (t == w1) {
                w1 = min(t + kMaskTiles, t1);
                const int lane = threadIdx.x & 63;
                const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
                lds_barrier();
                for (int i = t + wave; i < w1; i += waves) {
                    const int j = i * kKeyTile + lane;
                    const uint64_t v = __ballot(j < Lk && mask[j] != 0);
                    if (lane == 0) bits[i & (kMaskTiles - 1)] = v;
                }
                lds_barrier();
            }
            *kept = scalar64(bits[t & (kMaskTiles - 1)]);
            if (*kept != 0) return t;
        }
        *kept = 0;
        return t1;
    }
};

// Whether rows come in 16-byte chunks: what load_chunk's vec asks for, and with
// close_rows what direct loads to LDS do.
inline bool chunked(const void* p, const int64_t s[3], int D) {
    return D % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 8 == 0 &&
           s[1] % 8 == 0 && s[2] % 8 == 0;
}

// |scale| log2 e, or 1 for a scale of 0 (which makes the queries zeros).
inline float score_scale(const Attention& a) {
    return a.scale != 0 ? (a.scale < 0 ? -a.scale : a.scale) * 1.44269504088896341f : 1.0f;
}

// Where the running maximum of a row's scores starts: it stays finite times
// c = score_scale, so that a row (or the keys of it so far) without any score
// above -inf has exponentials of 0 and a sum of 0, not NaN.
inline float lowest_score(float c) { return -0x1p127f / (c > 1.0f ? c : 1.0f); }

inline bool close_rows(int64_t stride) { return stride >= 0 && stride < (1 << 23); }

}  // namespace nova
