// Linear layers on 16-bit operands (bf16 / fp16), fp32 accumulation on the matrix cores:
//
//   forward   z = x W^T + b,  y = resid + act(z)              (z kept in 16 bits for the backward pass)
//   backward  dz = g * act'(z),  dx = dz W,  dW = dz^T x,  db = colsum(dz)
//
// the mixed-precision form of the denoisers' nn.Linear + F.gelu (+ skip) layers (models/direction_diffusion.py:47-69,
// ddpm.py:9-27; the fp32 form is gemm_limbs.hip).  Bias, activation, residual and the copy of z leave the accumulators
// in fp32 and are rounded once each.  dz is rounded to the operands' type, as the matrix instruction needs it; db is
// summed from the unrounded products.
//
// One tile kernel does the three products C[m][n] = sum_k A(m, k) B(n, k).  They differ in which index of an operand is
// contiguous: k (x and W forward, dz for dx) or the other one (W for dx, dz and x for dW).  In the second case a tile
// lies in LDS as it does in memory, k rows of m or n, and gfx950's transposing LDS read (ds_read_b64_tr_b16) hands a lane
// four consecutive k of its own column, so nothing is transposed in memory.
//
//   staging   16-byte chunks go from memory to LDS without passing registers where every row starts on a 16-byte border and
//             holds whole chunks; otherwise (an odd width, a sliced matrix) through registers, with the tail masked.  Chunks
//             beyond the contraction's end come from a page of zeros, rows and columns beyond the matrix from a valid one
//             (their results are not stored).
//   LDS       a k-contiguous tile has rows of BK elements whose chunks are permuted by row (c ^ f(row)) so that the 16-byte
//             reads of a fragment meet 128 bytes of distinct banks per clock (measured: 7.8 clocks per 1 KB read, 16 without);
//             the rows of B are dealt to the fragment so that a lane ends with 8 consecutive n: 16-byte stores.
//   split     the contraction of dW (the rows of the batch) is cut into slices, one workgroup each; fp32 partial tiles are
//             summed in slice order by a second launch, which also finishes db: the same bits on every call.
#include <stdlib.h>
#include "hd_common.cuh"
#include "hd_half.cuh"
#include "hd_gelu.cuh"
#include "../../include/hypdiff.h"

using namespace hd;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

__device__ __attribute__((aligned(16))) const unsigned zero_page[4] = {0, 0, 0, 0};

template <typename T> __device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma<bf16>(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma<f16>(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ void dma16(const void* g, char* l) {              // the hardware adds 16 * lane to the wavefront's l
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// ---- one operand's tile in LDS ----------------------------------------------------------------------------------------------
// k-contiguous: MN rows of BK elements.  k-strided (TR): BK rows of MN elements.  Addresses in bytes.
template <int MN, int BK, bool TR, bool PERM>
struct Tile16 {
    static constexpr int kRowChunks = (TR ? MN : BK) / 8;
    static constexpr int kChunks = MN * BK / 8;
    static constexpr int kBytes = MN * BK * 2;
    static_assert(!TR || MN >= 32, "a k-strided row holds at least two 16-column groups");
    // chunk c of row r lies at position c ^ swz(r)
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (TR) {
            const int g = (r & 3) | ((r >> 3) & 1) << 2;
            return (g << 1) & (kRowChunks - 2);                              // pairs of chunks (one 16-column group) move together
        } else if constexpr (PERM) {
            return (((r >> 1) & 1) | ((r >> 3) & 3) << 1) & (kRowChunks - 1);
        } else {
            return (r >> 1) & (kRowChunks - 1);
        }
    }
    // fragment f (16 of MN) for k = 32 s .. + 31: lane (r16, kq) gets k = 8 kq .. + 7 of its row / column.  PERM deals the
    // rows so that fragments 2 p and 2 p + 1 hold 8 consecutive ones per group of four accumulators.
    static __device__ __forceinline__ int frag_row(int f, int r16) {
        if constexpr (PERM) return 32 * (f >> 1) + 8 * (r16 >> 2) + 4 * (f & 1) + (r16 & 3);
        else return 16 * f + r16;
    }
    // the lane's part of a fragment's address; the rest (frag_off) is a constant of (f, s)
    static __device__ __forceinline__ uint4 read(const char* lds, int base_mn, int f, int s, int lane) {
        const int r16 = lane & 15, kq = lane >> 4;
        if constexpr (!TR) {
            const int r = base_mn + frag_row(f, r16);
            return *reinterpret_cast<const uint4*>(lds + r * (BK * 2) + (((s * 4 + kq) ^ swz(r)) << 4));
        } else {
            // this lane names 4 columns of k row `rho` of its group; it receives column r16 of 4 rows, twice
            const int rho = r16 >> 2, gam = r16 & 3;
            const int col = base_mn + (PERM ? 32 * (f >> 1) + 8 * gam + 4 * (f & 1) : 16 * f + 4 * gam);
            const int k0 = 32 * s + 8 * kq + rho;
            const int c = col >> 3, b = (col & 4) << 1;
            const char* p0 = lds + k0 * (MN * 2) + ((c ^ swz(k0)) << 4) + b;
            const char* p1 = lds + (k0 + 4) * (MN * 2) + ((c ^ swz(k0 + 4)) << 4) + b;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p0);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p1);
            struct { s16x4 a, b; } v = {lo, hi};
            return __builtin_bit_cast(uint4, v);
        }
    }
};

// What a workgroup stages of one operand: chunk q (0 .. kChunks - 1) of every k slab
template <typename T, typename L, int NT, int MN, int BK, bool TR, bool DIRECT>
struct Stager {
    static constexpr int kPer = L::kChunks / NT;                              // chunks of a thread
    static_assert(L::kChunks % NT == 0, "whole rounds");
    const T* p[kPer];                                                         // the chunk of the slab at hand
    int k[kPer];                                                              // its first k (k-contiguous) or its k (k-strided)
    int n_ok[kPer];                                                           // registers path: elements inside the row (k-strided)
    uint4 reg[DIRECT ? 1 : kPer];
    long long step;
    int k_end;

    __device__ __forceinline__ void init(const T* base, long long ld, int mn0, int mn_end, int k0, int k_end_, int tid) {
        k_end = k_end_;
        step = TR ? (long long)BK * ld : BK;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            const int at = q * NT + tid, r = at / L::kRowChunks, c = (at % L::kRowChunks) ^ L::swz(r);
            if constexpr (TR) {
                k[q] = k0 + r;
                int col = mn0 + c * 8;
                n_ok[q] = mn_end - col;
                if (n_ok[q] <= 0) { col = 0; n_ok[q] = 0; }                   // beyond the matrix: any column
                p[q] = base + (long long)k[q] * ld + col;
            } else {
                k[q] = k0 + c * 8;
                int row = mn0 + r;
                if (row >= mn_end) row = mn_end - 1;                          // beyond the matrix: any row
                n_ok[q] = 0;
                p[q] = base + (long long)row * ld + k[q];
            }
        }
    }
    __device__ __forceinline__ void advance() {
#pragma unroll
        for (int q = 0; q < kPer; ++q) { p[q] += step; k[q] += BK; }
    }
    // DIRECT: the slab at hand goes to LDS (in flight); otherwise into registers, and store() brings it to LDS
    __device__ __forceinline__ void load(char* lds, int wave) {
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            if constexpr (DIRECT) {
                const void* src = k[q] < k_end ? (const void*)p[q] : (const void*)zero_page;   // whole chunks (k_end % 8 == 0, or a k row)
                dma16(src, lds + (q * NT + wave * 64) * 16);
            } else {
                Pack<T, 8> v;
                const int ok = TR ? (k[q] < k_end ? n_ok[q] : 0) : k_end - k[q];
                if (ok >= 8) {
                    v = load_pack<T, 8>(p[q]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v.v[e] = e < ok ? p[q][e] : (T)0.f;
                }
                reg[q] = __builtin_bit_cast(uint4, v);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int q = 0; q < kPer; ++q) *reinterpret_cast<uint4*>(lds + (q * NT + tid) * 16) = reg[q];
        }
    }
};

__device__ __forceinline__ float act_value(float z, int act) {
    return act == HD_ACT_GELU ? gelu_erfc(z) : (act == HD_ACT_RELU ? (z > 0.f ? z : (z != z ? z : 0.f)) : z);
}
__device__ __forceinline__ float act_slope(float z, int act) {
    return act == HD_ACT_GELU ? gelu_erf_grad(z) : (act == HD_ACT_RELU ? (z > 0.f ? 1.f : 0.f) : 1.f);
}

struct Prod {
    const void *A, *B;
    long long lda, ldb;
    int M, N, K;
    void* C;                        // T (M, N) with pitch ldc, or fp32 partial tiles [slice][M][N]
    long long ldc;
    const void *bias, *resid;
    void* z;                        // (M, N) contiguous
    long long ldr;
    int act;
    int tiles_n, tiles, total;      // total = tiles * slices
    int slabs, slabs_rem;           // slice s covers slabs + (s < slabs_rem) slabs of BK
};

// 8 consecutive n of one row m leave: bias, z, activation, residual, rounding
template <typename T>
__device__ __forceinline__ void write8(const Prod& g, int m, int n, const float (&acc)[8]) {
    float v[8];
    const bool whole = n + 8 <= g.N;
    const T* bias = (const T*)g.bias;
    const T* resid = (const T*)g.resid;
    const long long o = (long long)m * g.ldc + n;
    if (whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[e];
        if (bias) {
            const Pack<T, 8> b = load_pack<T, 8>(bias + n);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += (float)b.v[e];
        }
        if (g.z) {
            Pack<T, 8> zz;
#pragma unroll
            for (int e = 0; e < 8; ++e) zz.v[e] = (T)v[e];
            store_pack<T, 8>((T*)g.z + (long long)m * g.N + n, zz);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = act_value(v[e], g.act);
        if (resid) {
            const Pack<T, 8> r = load_pack<T, 8>(resid + (long long)m * g.ldr + n);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += (float)r.v[e];
        }
        Pack<T, 8> y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y.v[e] = (T)v[e];
        store_pack<T, 8>((T*)g.C + o, y);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (n + e >= g.N) break;
            float s = acc[e] + (bias ? (float)bias[n + e] : 0.f);
            if (g.z) ((T*)g.z)[(long long)m * g.N + n + e] = (T)s;
            s = act_value(s, g.act);
            if (resid) s += (float)resid[(long long)m * g.ldr + n + e];
            ((T*)g.C)[o + e] = (T)s;
        }
    }
}

__device__ __forceinline__ void write8_f32(float* c, int N, int m, int n, const float (&acc)[8]) {
    float* o = c + (long long)m * N + n;
    if (n + 8 <= N) {
        Pack<float, 4> a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) { a.v[e] = acc[e]; b.v[e] = acc[4 + e]; }
        store_pack<float, 4>(o, a);
        store_pack<float, 4>(o + 4, b);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < N) o[e] = acc[e];
    }
}

// ---- the tile kernel: 4 wavefronts as 2 x 2, two LDS buffers, one barrier a slab ------------------------------------------------
template <typename T, bool TA, bool TB, bool DIRECT, int BM, int BN, int BK, bool PARTIAL>
__device__ __forceinline__ void tile_item(const Prod& g, int vid, char* lds) {
    using LA = Tile16<BM, BK, TA, false>;
    using LB = Tile16<BN, BK, TB, true>;
    constexpr int kStage = LA::kBytes + LB::kBytes;
    constexpr int FI = BM / 32, FJ = BN / 32;                                 // fragments of a wavefront
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tile = vid % g.tiles, slice = vid / g.tiles;
    const int tm = tile / g.tiles_n, tn = tile - tm * g.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;
    const int nslab = g.slabs + (slice < g.slabs_rem ? 1 : 0);
    const int k0 = (slice * g.slabs + (slice < g.slabs_rem ? slice : g.slabs_rem)) * BK;
    Stager<T, LA, 256, BM, BK, TA, DIRECT> sa;
    Stager<T, LB, 256, BN, BK, TB, DIRECT> sb;
    sa.init((const T*)g.A, g.lda, m0, g.M, k0, g.K, tid);
    sb.init((const T*)g.B, g.ldb, n0, g.N, k0, g.K, tid);
    const int wr = wave >> 1, wc = wave & 1;
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    sa.load(lds, wave);
    sb.load(lds + LA::kBytes, wave);
    sa.store(lds, tid);
    sb.store(lds + LA::kBytes, tid);
    for (int t = 0; t < nslab; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                                      // slab t is in LDS; the other buffer is free
        char* cur = lds + (t & 1) * kStage;
        char* nxt = lds + ((t + 1) & 1) * kStage;
        if (t + 1 < nslab) {                                                  // in flight during the multiplies
            sa.advance();
            sb.advance();
            sa.load(nxt, wave);
            sb.load(nxt + LA::kBytes, wave);
        }
#pragma unroll
        for (int s = 0; s < BK / 32; ++s) {
            uint4 fa[FI], fb[FJ];
#pragma unroll
            for (int i = 0; i < FI; ++i) fa[i] = LA::read(cur, wr * (BM / 2), i, s, lane);
#pragma unroll
            for (int j = 0; j < FJ; ++j) fb[j] = LB::read(cur + LA::kBytes, wc * (BN / 2), j, s, lane);
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = mfma<T>(fb[j], fa[i], acc[i][j]);   // D rows = n, D columns = m
        }
        if (t + 1 < nslab) {
            sa.store(nxt, tid);
            sb.store(nxt + LA::kBytes, tid);
        }
    }
    const int r16 = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        const int m = m0 + wr * (BM / 2) + 16 * i + r16;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < FJ; j += 2) {
            const int n = n0 + wc * (BN / 2) + 16 * j + 8 * kq;
            if (n >= g.N) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = acc[i][j][e]; v[4 + e] = acc[i][j + 1][e]; }
            if constexpr (PARTIAL) write8_f32((float*)g.C + (long long)slice * g.M * g.N, g.N, m, n, v);
            else write8<T>(g, m, n, v);
        }
    }
}

template <typename T, bool TA, bool TB, bool DIRECT, int BM, int BN, int BK, bool PARTIAL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void half_gemm(const Prod g) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * (BM + BN) * BK * 2];
    // workgroup b runs on XCD b % 8: every XCD a contiguous run of (slice, tile) pairs, so that tiles sharing rows meet in one L2
    const int per_xcd = (gridDim.x + 7) >> 3;
    const int vid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (vid >= g.total) return;                                               // uniform: the grid is rounded up to a multiple of 8
    tile_item<T, TA, TB, DIRECT, BM, BN, BK, PARTIAL>(g, vid, lds);
}

// ---- dz = g * act'(z) and the column sums of the unrounded products --------------------------------------------------------------
// A thread owns 8 columns and every (256 / lanes)-th row of the workgroup's rows; part[workgroup][N] gets the sums.
template <typename T>
__global__ __launch_bounds__(256) void act_bwd_k(const T* __restrict__ g, long long ldg, const T* __restrict__ z, int M, int N, int act,
                                                 int log2_lanes, int rows_wg, int col_tiles, T* __restrict__ dz, float* __restrict__ part) {
    __shared__ float red[256 * 8];
    const int lanes = 1 << log2_lanes, slots = 256 >> log2_lanes;
    const int rb = blockIdx.x / col_tiles, ct = blockIdx.x - rb * col_tiles;
    const int n = (ct * lanes + (threadIdx.x & (lanes - 1))) * 8;
    const int slot = threadIdx.x >> log2_lanes;
    const int m0 = rb * rows_wg, m1 = M - m0 < rows_wg ? M : m0 + rows_wg;
    float s[8] = {};
    if (n < N) {
        const bool whole = n + 8 <= N;
        for (int m = m0 + slot; m < m1; m += slots) {
            Pack<T, 8> a, b;
            const T* gp = g + (long long)m * ldg + n;
            const T* zp = z + (long long)m * N + n;
            if (whole) {
                a = load_pack<T, 8>(gp);
                if (act != HD_ACT_IDENTITY) b = load_pack<T, 8>(zp);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a.v[e] = n + e < N ? gp[e] : (T)0.f;
                    b.v[e] = act != HD_ACT_IDENTITY && n + e < N ? zp[e] : (T)0.f;
                }
            }
            Pack<T, 8> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = act != HD_ACT_IDENTITY ? (float)a.v[e] * act_slope((float)b.v[e], act) : (float)a.v[e];
                s[e] += d;
                o.v[e] = (T)d;
            }
            if (dz) {
                T* p = dz + (long long)m * N + n;
                if (whole) {
                    store_pack<T, 8>(p, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n + e < N) p[e] = o.v[e];
                }
            }
        }
    }
    if (!part) return;                                                        // uniform
#pragma unroll
    for (int e = 0; e < 8; ++e) red[e * 256 + threadIdx.x] = s[e];
    __syncthreads();
    if (slot == 0 && n < N) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float t = 0.f;
            for (int q = 0; q < slots; ++q) t += red[e * 256 + q * lanes + threadIdx.x];
            if (n + e < N) part[(long long)rb * N + n + e] = t;
        }
    }
}

// ---- partial sums in order: dW from its slices, db from its row blocks -----------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void half_reduce_k(const float* __restrict__ ws, int nsl, long long count, T* __restrict__ dw, int w_wgs,
                                                     const float* __restrict__ part, int nparts, int N, T* __restrict__ db) {
    if ((int)blockIdx.x < w_wgs) {
        const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
        if (i >= count) return;
        if (i + 4 <= count) {
            Pack<float, 4> s = load_pack<float, 4>(ws + i);
#pragma unroll 4
            for (int k = 1; k < nsl; ++k) {
                const Pack<float, 4> a = load_pack<float, 4>(ws + k * count + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) s.v[e] += a.v[e];
            }
            Pack<T, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = (T)s.v[e];
            store_pack<T, 4>(dw + i, o);
        } else {
            for (long long j = i; j < count; ++j) {
                float s = ws[j];
                for (int k = 1; k < nsl; ++k) s += ws[k * count + j];
                dw[j] = (T)s;
            }
        }
        return;
    }
    __shared__ float red[16][16];                                             // 16 columns, 16 runs of row blocks each
    const int col = threadIdx.x & 15, run = threadIdx.x >> 4;
    const int n = ((int)blockIdx.x - w_wgs) * 16 + col;
    const int per = (nparts + 15) / 16, a = run * per, b = a + per < nparts ? a + per : nparts;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int k = a; k < b; ++k) s += part[(long long)k * N + n];
    }
    red[run][col] = s;
    __syncthreads();
    if (run == 0 && n < N) {
        for (int k = 1; k < 16; ++k) s += red[k][col];
        db[n] = (T)s;
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------------------
inline bool direct_ok(const void* p, int64_t ld, int64_t inner, int64_t outer) {
    return (uintptr_t)p % 16 == 0 && inner % 8 == 0 && (ld % 8 == 0 || outer == 1);
}

constexpr int kBM = 128, kBN = 128, kBK = 64;

template <typename T, bool TA, bool TB, bool PARTIAL>
void launch_product(Prod g, int slices, bool direct, hipStream_t st) {
    g.tiles_n = (g.N + kBN - 1) / kBN;
    g.tiles = (g.M + kBM - 1) / kBM * g.tiles_n;
    g.total = g.tiles * slices;
    const int slabs = (g.K + kBK - 1) / kBK;
    g.slabs = slabs / slices;
    g.slabs_rem = slabs % slices;
    const unsigned grid = (unsigned)((g.total + 7) / 8 * 8);
    if (direct) half_gemm<T, TA, TB, true, kBM, kBN, kBK, PARTIAL><<<grid, 256, 0, st>>>(g);
    else half_gemm<T, TA, TB, false, kBM, kBN, kBK, PARTIAL><<<grid, 256, 0, st>>>(g);
}

inline int dw_slices(int64_t R, int64_t P, int64_t Q) {
    // one resident round of two workgroups per CU; slices of at least two slabs
    const int64_t tiles = ((P + kBM - 1) / kBM) * ((Q + kBN - 1) / kBN);
    int64_t s = 512 / tiles;
    const int64_t most = (R + 2 * kBK - 1) / (2 * kBK);
    s = s > most ? most : s;
    return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

struct BwdPlan {
    int log2_lanes, col_tiles, rows_wg, row_wgs, slices;
    bool need_dz;
    int64_t off_part, off_ws, bytes;
};

BwdPlan bwd_plan(int64_t M, int64_t N, int64_t K, int act) {
    BwdPlan p;
    const int64_t groups = (N + 7) / 8;
    p.log2_lanes = 0;
    while (p.log2_lanes < 8 && (int64_t(1) << p.log2_lanes) < groups) ++p.log2_lanes;
    p.col_tiles = (int)((groups + (1 << p.log2_lanes) - 1) >> p.log2_lanes);
    const int slots = 256 >> p.log2_lanes;
    // about 1024 workgroups, at least 8 rows for a thread to sum
    int64_t rows = (M * p.col_tiles + 1023) / 1024;
    rows = rows < 8 * slots ? 8 * slots : rows;
    rows = (rows + slots - 1) / slots * slots;
    p.rows_wg = (int)rows;
    p.row_wgs = (int)((M + rows - 1) / rows);
    p.slices = dw_slices(M, N, K);
    p.need_dz = act != HD_ACT_IDENTITY;
    auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    int64_t at = p.need_dz ? up(M * N * 2) : 0;
    p.off_part = at;
    at += up((int64_t)p.row_wgs * N * 4);
    p.off_ws = at;
    at += up((int64_t)p.slices * N * K * 4);
    p.bytes = at > 256 ? at : 256;
    return p;
}

bool known_act(int a) { return a == HD_ACT_IDENTITY || a == HD_ACT_RELU || a == HD_ACT_GELU; }

#define HD_LINEAR_SHAPE(fn)                                                                                                     \
    HD_REQUIRE(dtype == HD_DT_BF16 || dtype == HD_DT_F16, fn ": element type bf16 or fp16, not %d", dtype);                      \
    HD_REQUIRE(known_act(act), fn ": activation identity, relu or gelu, not %d", act);                                          \
    HD_REQUIRE(M >= 0 && M < (1LL << 30) && N >= 1 && N < (1LL << 24) && K >= 1 && K < (1LL << 24), fn ": bad shape");             \
    HD_REQUIRE(ldx >= K && ldw >= K, fn ": row pitch below the width")

template <typename T>
int linear_fwd(const Prod& g, bool direct, hipStream_t s) {
    launch_product<T, false, false, false>(g, 1, direct, s);
    return check_launch("hd_linear_act_fwd");
}

template <typename T>
int linear_bwd(const T* g, int64_t ldg, const T* z, const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t M, int64_t N, int64_t K,
               int act, T* dx, T* dw, T* db, const BwdPlan& p, unsigned char* ws, hipStream_t s) {
    const T* dz = g;
    long long lddz = ldg;
    float* part = db ? (float*)(ws + p.off_part) : nullptr;
    if (p.need_dz || db) {
        T* o = p.need_dz && (dx || dw) ? (T*)ws : nullptr;
        act_bwd_k<T><<<(unsigned)(p.row_wgs * p.col_tiles), 256, 0, s>>>(g, ldg, z, (int)M, (int)N, act, p.log2_lanes, p.rows_wg, p.col_tiles,
                                                                        o, part);
        if (o) { dz = o; lddz = N; }
    }
    Prod q = {};
    q.act = HD_ACT_IDENTITY;
    if (dx) {                                                                 // (M, K) = dz (M, N) . W (N, K)
        q.A = dz; q.lda = lddz; q.B = w; q.ldb = ldw; q.M = (int)M; q.N = (int)K; q.K = (int)N; q.C = dx; q.ldc = K;
        launch_product<T, false, true, false>(q, 1, direct_ok(dz, lddz, N, M) && direct_ok(w, ldw, K, N), s);
    }
    if (dw) {                                                                 // (N, K) = dz^T (N, M) . x (M, K)
        q.A = dz; q.lda = lddz; q.B = x; q.ldb = ldx; q.M = (int)N; q.N = (int)K; q.K = (int)M; q.C = ws + p.off_ws; q.ldc = K;
        launch_product<T, true, true, true>(q, p.slices, direct_ok(dz, lddz, N, M) && direct_ok(x, ldx, K, M), s);
    }
    if (dw || db) {
        const int64_t count = dw ? N * K : 0;
        const int w_wgs = (int)((count + 1023) / 1024), b_wgs = db ? (int)((N + 15) / 16) : 0;
        half_reduce_k<T><<<(unsigned)(w_wgs + b_wgs), 256, 0, s>>>((const float*)(ws + p.off_ws), p.slices, count, dw, w_wgs, part, p.row_wgs,
                                                                   (int)N, db);
    }
    return check_launch("hd_linear_act_bwd");
}

}  // namespace

extern "C" int hd_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* resid, int64_t ldr,
                                 int dtype, int64_t M, int64_t N, int64_t K, int act, void* y, void* z, void* st) {
    HD_LINEAR_SHAPE("hd_linear_act_fwd");
    if (M == 0) return HD_OK;
    HD_REQUIRE(x && w && y, "hd_linear_act_fwd: null pointer");
    HD_REQUIRE(!resid || ldr >= 0, "hd_linear_act_fwd: negative pitch");
    HD_REQUIRE((((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)z | (uintptr_t)bias | (uintptr_t)resid) & 1) == 0,
               "hd_linear_act_fwd: pointer not aligned to the element");
    HD_REQUIRE(((M + kBM - 1) / kBM) * ((N + kBN - 1) / kBN) < (1LL << 31) - 8, "hd_linear_act_fwd: too many tiles");
    Prod g = {};
    g.A = x; g.lda = ldx; g.B = w; g.ldb = ldw; g.M = (int)M; g.N = (int)N; g.K = (int)K;
    g.C = y; g.ldc = N; g.bias = bias; g.resid = resid; g.ldr = ldr; g.z = z; g.act = act;
    const bool direct = direct_ok(x, ldx, K, M) && direct_ok(w, ldw, K, N);
    return dtype == HD_DT_BF16 ? linear_fwd<bf16>(g, direct, (hipStream_t)st) : linear_fwd<f16>(g, direct, (hipStream_t)st);
}

extern "C" int64_t hd_linear_act_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int act) {
    if (M < 0 || N < 1 || K < 1 || M >= (1LL << 30) || N >= (1LL << 24) || K >= (1LL << 24) || !known_act(act)) return 0;
    return bwd_plan(M, N, K, act).bytes;
}

extern "C" int hd_linear_act_bwd(const void* g, int64_t ldg, const void* z, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                 int dtype, int64_t M, int64_t N, int64_t K, int act, void* dx, void* dw, void* db, void* workspace,
                                 int64_t workspace_bytes, void* st) {
    HD_LINEAR_SHAPE("hd_linear_act_bwd");
    HD_REQUIRE(ldg >= N, "hd_linear_act_bwd: row pitch below the width");
    HD_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0, "hd_linear_act_bwd: null or misaligned workspace");
    HD_REQUIRE(M == 0 || (g && (z || act == HD_ACT_IDENTITY)), "hd_linear_act_bwd: null pointer");
    HD_REQUIRE(!(dx && M > 0) || w, "hd_linear_act_bwd: dx needs w");
    HD_REQUIRE(!(dw && M > 0) || x, "hd_linear_act_bwd: dw needs x");
    HD_REQUIRE((((uintptr_t)g | (uintptr_t)z | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db) & 1) == 0,
               "hd_linear_act_bwd: pointer not aligned to the element");
    HD_REQUIRE(M > 0, "hd_linear_act_bwd: no rows (the gradients are zeros; fill them)");
    const BwdPlan p = bwd_plan(M, N, K, act);
    HD_REQUIRE(workspace_bytes >= p.bytes, "hd_linear_act_bwd: workspace of %lld bytes required, got %lld", (long long)p.bytes,
               (long long)workspace_bytes);
    HD_REQUIRE(((M + kBM - 1) / kBM) * ((K + kBN - 1) / kBN) < (1LL << 31) - 8 &&
                   ((N + kBM - 1) / kBM) * ((K + kBN - 1) / kBN) * p.slices < (1LL << 31) - 8,
               "hd_linear_act_bwd: too many tiles");
    unsigned char* ws = (unsigned char*)workspace;
    hipStream_t s = (hipStream_t)st;
    if (dtype == HD_DT_BF16)
        return linear_bwd<bf16>((const bf16*)g, ldg, (const bf16*)z, (const bf16*)x, ldx, (const bf16*)w, ldw, M, N, K, act, (bf16*)dx,
                                (bf16*)dw, (bf16*)db, p, ws, s);
    return linear_bwd<f16>((const f16*)g, ldg, (const f16*)z, (const f16*)x, ldx, (const f16*)w, ldw, M, N, K, act, (f16*)dx, (f16*)dw,
                           (f16*)db, p, ws, s);
}
