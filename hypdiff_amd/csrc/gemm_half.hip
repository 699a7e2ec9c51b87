// Linear layers on 16-bit operands (bf16 / fp16), fp32 accumulation on the matrix cores:
//
//   forward   z = x W^T + b,  y = resid + act(z)              (z kept in fp16 for the backward pass)
//   backward  dz = g * act'(z),  dx = dz W,  dW = dz^T x,  db = colsum(dz)
//
// the mixed-precision form of the denoisers' nn.Linear + F.gelu (+ skip) layers (models/direction_diffusion.py:47-69,
// ddpm.py:9-27; the fp32 form is gemm_limbs.hip).  Bias, activation, residual and the copy of z leave the accumulators
// in fp32 and are rounded once each.  dz is rounded to the operands' type, as the matrix instruction needs it; db is
// summed from the unrounded products.
//
// Three products C[m][n] = sum_k A(m, k) B(n, k): forward (A = x, B = W), dx (A = dz, B = W^T, which the launch that makes dz
// also writes), dW (A = dz, B = x, both with k -- the rows of the batch -- as the slow index).
//
//   tiles     128 x 192, 128 x 128, 64 x 128 or 64 x 64 of 4 wavefronts, by a cost model (choose_tiles); 32 x 32 with the
//             contraction split over the wavefronts for few rows (small_gemm); dW 192 x 192 or 64 x 64 (dw_plan).  One slab of 64 k in LDS,
//             not two: a workgroup waits for its loads, and the 3 to 8 that fit a CU because of it multiply meanwhile.  Two
//             slabs, the next one's loads in flight during the multiplies, are no faster at any size (with a GELU of four
//             operations less an element, 74750 x 800 -> 900: 128 x 192 146 us, with two 155; 128 x 128 158 and 175;
//             4096 x 800 -> 900: 14.1 and 14.2 at 64 x 128), three slower.
//   staging   16-byte chunks go from memory to LDS without passing registers where every row starts on a 16-byte border and
//             holds whole chunks; otherwise (an odd width, a sliced matrix) through registers, with the tail masked.  Chunks
//             beyond the contraction's end come from a page of zeros, rows and columns beyond the matrix from a valid one
//             (their results are not stored).
//   LDS       a slab with k fast has rows of 128 or 64 bytes whose chunks are permuted by row (c ^ f(row)): a fragment's 16-byte reads
//             then meet distinct banks (measured 8 clocks per 1 KB, the port's width).  B's rows are dealt to the fragments
//             so that a lane ends with 6 neighbouring n and 16 neighbouring lanes with one row's 96: whole runs of 192 bytes
//             leave with one store (per-lane 16-byte pieces of 16 rows cost 60 us more at 74750 x 800 -> 900).  A slab with
//             k slow lies in LDS as it does in memory; gfx950's transposing read (ds_read_b64_tr_b16) hands a lane four
//             consecutive k of its own column, so nothing is transposed in memory.
//   split     the contraction of dW is cut into slices, one workgroup each; fp32 partial tiles are summed in slice order by
//             the last launch, which also finishes db: the same bits on every call.
// What bounds the large forward (74750 x 800 -> 900, bf16: 142 to 155 us): no unit alone.  By its counters the matrix pipe is busy
// 39 % of the cycles, the vector unit issues in 54 % (dx, without GELU, in 29 %), 2.2 GB of L2 lines reach the CUs (15 TB/s; a third
// more than the operands' bytes, as runs of 128 bytes of 1600-byte rows straddle lines), and 36 % of the wavefronts' time is
// waiting: the phases of a workgroup (loads, products, write-out) alternate, and the three of a CU overlap them in part.
#include <math.h>
#include <type_traits>
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

// Loads through a pointer that may be the zero page: named as global memory, or the compiler takes them for flat loads, which
// the waits for LDS reads then wait for too
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 global16(const void* p) { return *(const __attribute__((address_space(1))) u32x4_any*)p; }
__device__ __forceinline__ void dma16(const void* g, char* l) {              // the hardware adds 16 * lane to the wavefront's l
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// ---- one operand's slab in LDS ----------------------------------------------------------------------------------------------
// k fast: MN rows of BK elements.  k slow (TR): BK rows of MN elements.  Chunks of 8 elements, addresses in bytes.
template <int MN, int BK, bool TR>
struct Slab {
    static constexpr int kRowChunks = (TR ? MN : BK) / 8;
    static constexpr int kChunks = MN * BK / 8;
    static constexpr int kBytes = MN * BK * 2;
    // chunk c of row r lies at position c ^ swz(r)
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (!TR) return (r >> 1) & (kRowChunks - 1);
        // pairs of chunks (16 columns) move together; rows r and r + 8 of a half-wavefront must not meet
        else if constexpr (MN % 128 == 0) return ((r & 3) | ((r >> 3) & 1) << 2) << 1;
        else return (((r >> 1) & 1) | ((r >> 3) & 1) << 1) << 1;               // 192, 64: rows are 128 bytes off a 256-byte border
    }
    // fragment f (16 of MN from base_mn on), k = 32 s .. + 31: lane (r16, kq) gets k = 8 kq .. + 7 of row / column r16
    static __device__ __forceinline__ uint4 read(const char* lds, int base_mn, int f, int s, int lane) {
        const int r16 = lane & 15, kq = lane >> 4;
        if constexpr (!TR) {
            const int r = base_mn + 16 * f + r16;
            return *reinterpret_cast<const uint4*>(lds + r * (BK * 2) + (((s * 4 + kq) ^ swz(r)) << 4));
        } else {
            // this lane names 4 columns of k row `rho` of its group; it receives column r16 of 4 rows, twice
            const int rho = r16 >> 2, gam = r16 & 3;
            const int col = base_mn + 16 * f + 4 * gam, c = col >> 3, b = (col & 4) << 1;
            const int k0 = 32 * s + 8 * kq + rho;
            const char* p0 = lds + k0 * (MN * 2) + ((c ^ swz(k0)) << 4) + b;
            const char* p1 = lds + (k0 + 4) * (MN * 2) + ((c ^ swz(k0 + 4)) << 4) + b;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p0);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p1);
            struct { s16x4 a, b; } v = {lo, hi};
            return __builtin_bit_cast(uint4, v);
        }
    }
};

__device__ __forceinline__ u32x4 shift_out(u32x4 v, int n) {                  // drops the first n of 8 elements, zeros behind; 0 <= n < 8
    unsigned long long lo = ((unsigned long long)v[1] << 32) | v[0], hi = ((unsigned long long)v[3] << 32) | v[2];
    if (n >= 4) { lo = hi; hi = 0; }
    const int b = 16 * (n & 3);
    lo = (lo >> b) | (b ? hi << (64 - b) : 0ull);
    hi >>= b;
    return u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}

// What a workgroup stages of one operand: chunk q (0 .. kChunks - 1) of every slab.  DEAL > 0: the rows of a wavefront's DEAL rows
// lie in LDS in the order in which the fragments take them (fragment f, row r16 = row r16 * DEAL / 16 + f).
//
// Without DIRECT a chunk may start anywhere and the last one of a row (of 8 elements at least) may be short: then the row's last 8
// elements are loaded and shifted into place on the way to LDS.  No lane branches around a load (a branch per chunk kept the
// loads from being in flight together: dW of 7850 x 800 x 513 28 us against 21).
template <typename T, int MN, int BK, bool TR, bool DIRECT, int DEAL>
struct Stager {
    using L = Slab<MN, BK, TR>;
    static constexpr int kPer = L::kChunks / 256;                             // chunks of a thread
    static_assert(L::kChunks % 256 == 0, "whole rounds");
    // k fast: a thread's chunks lie in rows 256 / kRowChunks apart, at one position and, as swz() repeats by then, of one k
    static_assert(TR || (256 % L::kRowChunks == 0 && 256 / L::kRowChunks % 16 == 0), "one k for all chunks of a thread");
    static constexpr int kKs = TR ? kPer : 1;
    const T* p[kPer];                                                         // the chunk of the slab at hand
    int k[kKs];                                                               // its first k (k fast) or its k (k slow)
    int off[!DIRECT && TR ? kPer : 1];                                        // elements that its load starts early
    u32x4 reg[DIRECT ? 1 : kPer];
    long long step;
    int k_end;
    bool edge;                                                                // uniform: some chunk of the slab at hand is short

    static __device__ __forceinline__ int row_of(int r) {
        if constexpr (DEAL == 0) return r;
        else return r / DEAL * DEAL + (r % 16) * (DEAL / 16) + (r % DEAL) / 16;
    }
    __device__ __forceinline__ void init(const T* base, long long ld, int mn0, int mn_end, int k0, int k_end_, int tid) {
        k_end = k_end_;
        step = TR ? (long long)BK * ld : BK;
        edge = TR && mn0 + MN > mn_end;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            const int at = q * 256 + tid, r = at / L::kRowChunks, c = (at % L::kRowChunks) ^ L::swz(r);
            if constexpr (TR) {
                k[q] = k0 + r;
                int col = mn0 + c * 8;
                if (col >= mn_end) col = 0;                                   // beyond the matrix: any column
                if constexpr (!DIRECT) {
                    off[q] = col + 8 > mn_end ? col + 8 - mn_end : 0;
                    col -= off[q];
                }
                p[q] = base + (long long)k[q] * ld + col;
            } else {
                if (q == 0) k[0] = k0 + c * 8;
                int row = mn0 + row_of(r);
                if (row >= mn_end) row = mn_end - 1;                          // beyond the matrix: any row
                p[q] = base + (long long)row * ld + k[0];
            }
        }
    }
    __device__ __forceinline__ void advance() {
#pragma unroll
        for (int q = 0; q < kPer; ++q) p[q] += step;
#pragma unroll
        for (int q = 0; q < kKs; ++q) k[q] += BK;
    }
    // DIRECT: the slab at hand (from k_slab on) goes to LDS, in flight; otherwise into registers, and store() brings it to LDS
    __device__ __forceinline__ void load(char* lds, int wave, int k_slab) {
        if constexpr (DIRECT) {
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const void* src = k[TR ? q : 0] < k_end ? (const void*)p[q] : (const void*)zero_page;   // whole chunks, or a k row
                dma16(src, lds + (q * 256 + wave * 64) * 16);
            }
        } else {
            int early = 0;
            if constexpr (!TR) {
                edge = k_slab + BK > k_end;
                early = edge && k[0] + 8 > k_end ? k[0] + 8 - k_end : 0;
                off[0] = early & 7;
            }
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const T* src = k[TR ? q : 0] < k_end ? p[q] - early : (const T*)zero_page;
                reg[q] = global16(src);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) {
        if constexpr (!DIRECT) {
            if (edge) {
#pragma unroll
                for (int q = 0; q < kPer; ++q) reg[q] = shift_out(reg[q], off[TR ? q : 0]);
            }
#pragma unroll
            for (int q = 0; q < kPer; ++q) *reinterpret_cast<u32x4*>(lds + (q * 256 + tid) * 16) = reg[q];
        }
    }
};

// 2^SHIFT * 0.5 erfc(a / sqrt 2) for a = |x|, as 2^(a P(a) - 1 + SHIFT): a weighted minimax fit of log2 erfc.  Degree 8, so that
// GELU's negative tail is right to a quarter of the half step of the type it is rounded to: relative error 5.5e-5 down to x = -6, where
// fp16 ends, 3.3e-4 down to -13.3, where bf16 does (a degree of 4 is off by 0.4 % at -4 and by 17 % at -6), and 1.4e-6 |x| anywhere.
// Beyond 30 it is 0 in any case; the clamp keeps infinities out of the products.
template <int SHIFT>
__device__ __forceinline__ float half_erfc16(float x) {
    const float a = fminf(fabsf(x), 30.f);
    float r = fmaf(-1.26476807e-09f, a, 1.06469543e-07f);
    r = fmaf(r, a, -3.80471897e-06f);
    r = fmaf(r, a, 7.67703314e-05f);
    r = fmaf(r, a, -9.83094680e-04f);
    r = fmaf(r, a, 8.56748410e-03f);
    r = fmaf(r, a, -5.38930967e-02f);
    r = fmaf(r, a, -4.58624214e-01f);
    r = fmaf(r, a, -1.15118206e+00f);
    return __builtin_amdgcn_exp2f(fmaf(r, a, (float)(SHIFT - 1)));
}
// GELU(x) = (x + |x|) / 2 - |x| * (0.5 erfc(|x| / sqrt 2)); the first term passes a NaN on and +inf through.  The second is
// formed 2^24 above its value and brought down last: exp2 returns 0 below 2^-126, which x = -12.9 reaches
__device__ __forceinline__ float gelu16(float x) {
    return fmaf(fminf(fabsf(x), 30.f) * half_erfc16<24>(x), -0x1p-24f, fmaf(0.5f, fabsf(x), 0.5f * x));
}
// Phi(x) + x phi(x); Phi of a negative x without a difference that would round at 2^-25
__device__ __forceinline__ float gelu16_slope(float x) {
    const float q = half_erfc16<0>(x), Phi = x < 0.f ? q : 1.0f - q;
    return fmaf(x, __builtin_amdgcn_exp2f(fmaf(x * -0.72134752044448170368f, x, -1.32574806473615f)), Phi);   // log2(1 / sqrt(2 pi))
}
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == HD_ACT_GELU) return gelu16(z);
    else if constexpr (ACT == HD_ACT_RELU) return z > 0.f ? z : (z == z ? 0.f : z);
    else return z;
}
// g * act'(z).  ReLU selects: an infinite g under a closed unit leaves 0, and a NaN z passes g on
template <int ACT>
__device__ __forceinline__ float through_act(float g, float z) {
    if constexpr (ACT == HD_ACT_GELU) return g * gelu16_slope(z);
    else if constexpr (ACT == HD_ACT_RELU) return z <= 0.f ? 0.f : g;
    else return g;
}

// The pre-activation as it is kept for the backward pass: in fp16 for bf16 operands too, whose own 8 bits would add a third of dz's
// rounding to the gradients (error 1.5 instead of 1.41 roundings; for fp16 operands it is 1.47).  Only the slope reads it: beyond
// 30000 that is 0 or 1 (the clamp keeps fp16 finite), and a positive z stays positive for ReLU.  A NaN stays one.
__device__ __forceinline__ f16 kept_z(float z) {
    const float c = fminf(fmaxf(z, -30000.f), 30000.f);
    const float p = z > 0.f ? fmaxf(c, 0x1p-24f) : c;
    return (f16)(z == z ? p : z);
}

struct Prod {
    const void *A, *B;
    long long lda, ldb;
    int M, N, K;
    void* C;                        // T (M, N) contiguous, or fp32 partial tiles [slice][M][N]
    const void *bias, *resid;
    void* z;                        // fp16 (M, N) contiguous, or null
    long long ldr;
    int act;
    int z_past;                     // store z past the caches
    int tiles_n, tiles, total;      // total = tiles * slices
    int slabs, slabs_rem;           // slice s covers slabs + (s < slabs_rem) slabs of BK
};

// V neighbouring n of row m leave: bias, z, activation, residual, one rounding.  yb / zb: the tile's first element, off: this lane's
// byte offset in the tile.
template <typename T, int V, int ACT>
__device__ __forceinline__ void write_row(const Prod& g, char* yb, char* zb, unsigned off, int m, int n, const float (&acc)[V],
                                          const float (&bias)[V]) {
    float v[V];
    const T* resid = (const T*)g.resid + (long long)m * g.ldr + n;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = acc[e] + bias[e];
    if (n + V <= g.N) {
        if (zb) {
            Pack<f16, V> zz;
#pragma unroll
            for (int e = 0; e < V; ++e) zz.v[e] = kept_z(v[e]);
            if constexpr (V % 2 == 0) {
                typedef unsigned words __attribute__((ext_vector_type(V / 2), aligned(2)));
                words w;
                __builtin_memcpy(&w, &zz, sizeof(zz));
                if (g.z_past) __builtin_nontemporal_store(w, (words*)(zb + off));
                else __builtin_memcpy(zb + off, &w, sizeof(w));
            } else {
                store_pack<f16, V>((f16*)(zb + off), zz);
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = act_value<ACT>(v[e]);
        if (g.resid) {
            const Pack<T, V> r = load_pack<T, V>(resid);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += (float)r.v[e];
        }
        Pack<T, V> y;
#pragma unroll
        for (int e = 0; e < V; ++e) y.v[e] = (T)v[e];
        store_pack<T, V>((T*)(yb + off), y);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (n + e >= g.N) break;
            if (zb) ((f16*)(zb + off))[e] = kept_z(v[e]);
            float s = act_value<ACT>(v[e]);
            if (g.resid) s += (float)resid[e];
            ((T*)(yb + off))[e] = (T)s;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void load_bias(const Prod& g, int n, float (&bias)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = g.bias && n + e < g.N ? (float)((const T*)g.bias)[n + e] : 0.f;
}

// a wavefront's accumulators: D rows (4 kq + e) = m, D columns (r16), fragment by fragment = neighbouring n of lane r16
template <typename T, int FI, int FJ, int ACT>
__device__ __forceinline__ void write_tile(const Prod& g, const f32x4 (&acc)[FI][FJ], int m0, int n0, int lane) {
    const int r16 = lane & 15, kq = lane >> 4, n = n0 + r16 * FJ;
    float bias[FJ];
    load_bias<T, FJ>(g, n, bias);
    char* yb = (char*)g.C + ((long long)m0 * g.N + n0) * 2;
    char* zb = g.z ? (char*)g.z + ((long long)m0 * g.N + n0) * 2 : nullptr;
    const unsigned off = (unsigned)(kq * 4 * g.N + r16 * FJ) * 2;             // below 2^32: at most 128 rows, N < 2^23
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + 16 * i + 4 * kq + e;
            float v[FJ];
#pragma unroll
            for (int j = 0; j < FJ; ++j) v[j] = acc[i][j][e];
            if (m < g.M && n < g.N) write_row<T, FJ, ACT>(g, yb, zb, off + (unsigned)((16 * i + e) * g.N) * 2, m, n, v, bias);
        }
}

// ---- the tile kernel: 4 wavefronts as 2 x 2, one slab in LDS -------------------------------------------------------------------------
template <bool TR, bool DIRECT, int BM, int BN, int BK>
constexpr int kTileLds = (Slab<BM, BK, TR>::kBytes + Slab<BN, BK, TR>::kBytes);

template <typename T, bool TR, bool DIRECT, int BM, int BN, int BK>
__device__ __forceinline__ void tile_item(const Prod& g, int vid, char* lds) {
    constexpr int WM = BM / 2, WN = BN / 2, FI = WM / 16, FJ = WN / 16;       // a wavefront's part, its fragments
    using SA = Stager<T, BM, BK, TR, DIRECT, 0>;
    using SB = Stager<T, BN, BK, TR, DIRECT, TR ? 0 : WN>;
    constexpr int kA = SA::L::kBytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile = vid % g.tiles, slice = vid / g.tiles;
    const int tm = tile / g.tiles_n, tn = tile - tm * g.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;
    const int nslab = g.slabs + (slice < g.slabs_rem ? 1 : 0);
    const int k0 = (slice * g.slabs + (slice < g.slabs_rem ? slice : g.slabs_rem)) * BK;
    SA sa;
    SB sb;
    sa.init((const T*)g.A, g.lda, m0, TR ? (g.M + 7) / 8 * 8 : g.M, k0, g.K, tid);   // TR: dz, whose rows are whole chunks
    sb.init((const T*)g.B, g.ldb, n0, g.N, k0, g.K, tid);
    const int wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    sa.load(lds, wave, k0);                                                   // DIRECT: on its way to LDS; otherwise to registers
    sb.load(lds + kA, wave, k0);
    for (int t = 0; t < nslab; ++t) {
        sa.store(lds, tid);
        sb.store(lds + kA, tid);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                                      // slab t is in LDS
        if (!DIRECT && t + 1 < nslab) {                                       // to registers during the multiplies
            sa.advance();
            sb.advance();
            sa.load(lds, wave, k0 + (t + 1) * BK);
            sb.load(lds + kA, wave, k0 + (t + 1) * BK);
        }
#pragma unroll
        for (int s = 0; s < BK / 32; ++s) {
            uint4 fa[FI], fb[FJ];
#pragma unroll
            for (int i = 0; i < FI; ++i) fa[i] = SA::L::read(lds, wm, i, s, lane);
#pragma unroll
            for (int j = 0; j < FJ; ++j) fb[j] = SB::L::read(lds + kA, wn, j, s, lane);
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = mfma<T>(fa[i], fb[j], acc[i][j]);   // D rows = m, D columns = n
        }
        if (t + 1 < nslab) {
            __syncthreads();                                                  // every wavefront has read slab t
            if (DIRECT) {
                sa.advance();
                sb.advance();
                sa.load(lds, wave, k0 + (t + 1) * BK);
                sb.load(lds + kA, wave, k0 + (t + 1) * BK);
            }
        }
    }
    if constexpr (TR) {                                                       // fp32 partial tile of this slice
        const int r16 = lane & 15, kq = lane >> 4;
        float* o = (float*)g.C + (long long)slice * g.M * g.N;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + wm + 16 * i + 4 * kq + e;
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    const int n = n0 + wn + 16 * j + r16;
                    if (m < g.M && n < g.N) o[(long long)m * g.N + n] = acc[i][j][e];
                }
            }
    } else {
        if (g.act == HD_ACT_GELU) write_tile<T, FI, FJ, HD_ACT_GELU>(g, acc, m0 + wm, n0 + wn, lane);
        else if (g.act == HD_ACT_RELU) write_tile<T, FI, FJ, HD_ACT_RELU>(g, acc, m0 + wm, n0 + wn, lane);
        else write_tile<T, FI, FJ, HD_ACT_IDENTITY>(g, acc, m0 + wm, n0 + wn, lane);
    }
}

// OCC: wavefronts a SIMD that the registers have to allow, i.e. workgroups a CU
template <typename T, bool TR, bool DIRECT, int BM, int BN, int BK, int OCC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(OCC))) void half_gemm(const Prod g) {
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<TR, DIRECT, BM, BN, BK>];
    // workgroup b runs on XCD b % 8: every XCD a contiguous run of (slice, tile) pairs, so that tiles sharing rows meet in one L2
    const int per_xcd = (gridDim.x + 7) >> 3;
    const int vid = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (vid >= g.total) return;                                               // uniform: the grid is rounded up to a multiple of 8
    tile_item<T, TR, DIRECT, BM, BN, BK>(g, vid, lds);
}

// ---- few rows: 32 x 32 tiles, the contraction dealt over the 4 wavefronts -----------------------------------------------------------
// With so few tiles a slab-by-slab loop is a chain of load latencies (200 x 512 x 512: 8 workgroups of 16 slabs).  Here a
// wavefront loads the fragments of 4 slabs straight into registers, all in flight together, and multiplies; the four partial
// tiles meet in LDS, in wavefront order.  Any alignment: a fragment is 8 consecutive k of a row.
template <typename T>
__device__ __forceinline__ uint4 load_frag_tail(const T* row, int k, int K) {   // the slab that holds the row's end: zeros behind it
    Pack<T, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const T x = row[k + e < K ? k + e : K - 1];                           // no branch: the loads stay in flight together
        v.v[e] = k + e < K ? x : (T)0.f;
    }
    return __builtin_bit_cast(uint4, v);
}

constexpr int kSmallLds = 4 * 32 * 36 * 4;

template <typename T>
__device__ __forceinline__ void small_item(const Prod& g, int vid, char* lds) {
    float (*red)[32][36] = reinterpret_cast<float (*)[32][36]>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int tm = vid / g.tiles_n, tn = vid - tm * g.tiles_n;
    const int m0 = tm * 32, n0 = tn * 32;
    const T *pa[2], *pb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {                                             // beyond the matrix: any row
        const int m = m0 + 16 * i + r16 < g.M ? m0 + 16 * i + r16 : g.M - 1, n = n0 + 16 * i + r16 < g.N ? n0 + 16 * i + r16 : g.N - 1;
        pa[i] = (const T*)g.A + (long long)m * g.lda;
        pb[i] = (const T*)g.B + (long long)n * g.ldb;
    }
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int slabs = (g.K + 31) / 32;
    const int inside = g.K / 32;                                              // slabs without the row's end
    int t = wave;
    for (; t + 12 < inside; t += 16) {                                        // slabs t, t + 4, t + 8, t + 12
        uint4 fa[4][2], fb[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = (t + 4 * u) * 32 + 8 * kq;
                fa[u][i] = __builtin_bit_cast(uint4, load_pack<T, 8>(pa[i] + k));
                fb[u][i] = __builtin_bit_cast(uint4, load_pack<T, 8>(pb[i] + k));
            }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma<T>(fa[u][i], fb[u][j], acc[i][j]);
    }
    for (; t < slabs; t += 4) {                                               // the last few, one at a time
        uint4 fa[2], fb[2];
        const int k = t * 32 + 8 * kq;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (t < inside) {                                                 // uniform
                fa[i] = __builtin_bit_cast(uint4, load_pack<T, 8>(pa[i] + k));
                fb[i] = __builtin_bit_cast(uint4, load_pack<T, 8>(pb[i] + k));
            } else {
                fa[i] = load_frag_tail<T>(pa[i], k, g.K);
                fb[i] = load_frag_tail<T>(pb[i], k, g.K);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mfma<T>(fa[i], fb[j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][16 * i + 4 * kq + e][16 * j + r16] = acc[i][j][e];
    __syncthreads();
    const int r = tid >> 3, c = (tid & 7) * 4, m = m0 + r, n = n0 + c;
    if (m >= g.M || n >= g.N) return;
    float v[4], bias[4];
    load_bias<T, 4>(g, n, bias);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ((red[0][r][c + e] + red[1][r][c + e]) + red[2][r][c + e]) + red[3][r][c + e];
    char* yb = (char*)g.C + ((long long)m * g.N + n) * 2;
    char* zb = g.z ? (char*)g.z + ((long long)m * g.N + n) * 2 : nullptr;
    if (g.act == HD_ACT_GELU) write_row<T, 4, HD_ACT_GELU>(g, yb, zb, 0, m, n, v, bias);
    else if (g.act == HD_ACT_RELU) write_row<T, 4, HD_ACT_RELU>(g, yb, zb, 0, m, n, v, bias);
    else write_row<T, 4, HD_ACT_IDENTITY>(g, yb, zb, 0, m, n, v, bias);
}

template <typename T>
__global__ __launch_bounds__(256) void small_gemm(const Prod g) {
    __shared__ __attribute__((aligned(16))) char lds[kSmallLds];
    small_item<T>(g, (int)blockIdx.x, lds);
}

// dx by small_gemm and dW's slices by 64 x 64 tiles in one launch: with few rows neither fills the chip nor waits for the other
template <typename T, bool DIRECT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void small_pair(const Prod dx, const Prod dw, int dx_wgs) {
    constexpr int kTile = kTileLds<true, DIRECT, 64, 64, 64>;
    __shared__ __attribute__((aligned(1024))) char lds[kTile > kSmallLds ? kTile : kSmallLds];
    if ((int)blockIdx.x < dx_wgs) small_item<T>(dx, (int)blockIdx.x, lds);
    else tile_item<T, true, DIRECT, 64, 64, 64>(dw, (int)blockIdx.x - dx_wgs, lds);
}

// ---- dz = g * act'(z), the column sums of the unrounded products, and W^T ---------------------------------------------------------
// A thread owns 8 columns and every (256 / lanes)-th row of the workgroup's rows, four rows in flight; part[row block][N] gets
// the sums.  dz has the row pitch lddz, a multiple of 64, and zeros up to the next multiple of 8 columns, so that the products
// take whole chunks.  The workgroups behind transpose W (N, K) into wt (K, N) with the same pitch and padding; the last ones copy
// an x of fewer than 8 columns into rows of 8.
// n: the thread's first column.  WIDE (N >= 8): the thread of the last, short group takes the last 8 columns, of which
// some belong to its neighbour: those come out twice, equal, and are summed once; it also writes the zeros behind column N.
template <typename T, int ACT, bool WIDE>
__device__ __forceinline__ void dz_rows(const T* __restrict__ g, long long ldg, const f16* __restrict__ z, int N, int n, int m, int m1, int slots,
                                        T* __restrict__ dz, long long lddz, float (&s)[8]) {
    constexpr int U = 4;
    auto fetch = [&](auto* p) {
        using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        Pack<E, 8> v;
        if constexpr (WIDE) {
            v = load_pack<E, 8>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = n + e < N ? p[e] : (E)0.f;
        }
        return v;
    };
    const int pads = WIDE && dz && n + 8 == N ? (8 - N % 8) % 8 : 0;
    for (; m < m1; m += U * slots) {
        Pack<T, 8> a[U];
        Pack<f16, 8> b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = m + u * slots < m1 ? m + u * slots : m;              // a row that is not there: read another, count none
            a[u] = fetch(g + (long long)r * ldg + n);
            if constexpr (ACT != HD_ACT_IDENTITY) b[u] = fetch(z + (long long)r * N + n);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (m + u * slots >= m1) break;
            Pack<T, 8> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float d = (float)a[u].v[e];
                if constexpr (ACT != HD_ACT_IDENTITY) d = through_act<ACT>(d, (float)b[u].v[e]);
                s[e] += d;
                o.v[e] = (T)d;
            }
            if (dz) {
                T* out = dz + (long long)(m + u * slots) * lddz + n;
                store_pack<T, 8>(out, o);                                     // not WIDE: g = z = 0 behind N, so dz = 0
                for (int e = 0; e < pads; ++e) out[8 + e] = (T)0.f;
            }
        }
    }
}

template <typename T, int ACT>
__device__ __forceinline__ void dz_block(const T* __restrict__ g, long long ldg, const f16* __restrict__ z, int M, int N, int log2_lanes,
                                         int rows_wg, int col_tiles, T* __restrict__ dz, long long lddz, float* __restrict__ part,
                                         float* red) {
    const int lanes = 1 << log2_lanes, slots = 256 >> log2_lanes;
    const int rb = blockIdx.x / col_tiles, ct = blockIdx.x - rb * col_tiles;
    const int n = (ct * lanes + (threadIdx.x & (lanes - 1))) * 8;
    const int slot = threadIdx.x >> log2_lanes;
    const int m0 = rb * rows_wg, m1 = M - m0 < rows_wg ? M : m0 + rows_wg;
    float s[8] = {};
    int skip = 0;                                                             // columns before the thread's own
    if (n < N) {
        if (N >= 8) {
            skip = n + 8 <= N ? 0 : n + 8 - N;
            dz_rows<T, ACT, true>(g, ldg, z, N, n - skip, m0 + slot, m1, slots, dz, lddz, s);
        } else {
            dz_rows<T, ACT, false>(g, ldg, z, N, n, m0 + slot, m1, slots, dz, lddz, s);
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
            if (e >= skip && n - skip + e < N) part[(long long)rb * N + n - skip + e] = t;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void act_bwd_k(const T* __restrict__ g, long long ldg, const f16* __restrict__ z, int M, int N, int act,
                                                 int log2_lanes, int rows_wg, int col_tiles, int dz_wgs, T* __restrict__ dz, long long lddz,
                                                 float* __restrict__ part, const T* __restrict__ w, long long ldw, int K, T* __restrict__ wt, int wt_wgs,
                                                 const T* __restrict__ x, long long ldx, T* __restrict__ x8) {
    __shared__ float red[256 * 8];
    if ((int)blockIdx.x < dz_wgs) {
        if (act == HD_ACT_GELU) dz_block<T, HD_ACT_GELU>(g, ldg, z, M, N, log2_lanes, rows_wg, col_tiles, dz, lddz, part, red);
        else if (act == HD_ACT_RELU) dz_block<T, HD_ACT_RELU>(g, ldg, z, M, N, log2_lanes, rows_wg, col_tiles, dz, lddz, part, red);
        else dz_block<T, HD_ACT_IDENTITY>(g, ldg, z, M, N, log2_lanes, rows_wg, col_tiles, dz, lddz, part, red);
        return;
    }
    const int b = (int)blockIdx.x - dz_wgs;
    if (b >= wt_wgs) {                                                        // rows of fewer than 8 elements, zeros behind them
        const int m = (b - wt_wgs) * 256 + (int)threadIdx.x;
        if (m >= M) return;
        Pack<T, 8> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = e < K ? x[(long long)m * ldx + e] : (T)0.f;
        store_pack<T, 8>(x8 + (long long)m * 8, v);
        return;
    }
    T* tile = (T*)red;                                                        // 32 x 33
    const int tk = (K + 31) / 32, n0 = b / tk * 32, k0 = b % tk * 32;
    const int c = threadIdx.x & 31, r0 = threadIdx.x >> 5;
#pragma unroll
    for (int r = r0; r < 32; r += 8) tile[r * 33 + c] = n0 + r < N && k0 + c < K ? w[(long long)(n0 + r) * ldw + k0 + c] : (T)0.f;
    __syncthreads();
#pragma unroll
    for (int r = r0; r < 32; r += 8)
        if (k0 + r < K && n0 + c < (N + 7) / 8 * 8) wt[(long long)(k0 + r) * lddz + n0 + c] = tile[c * 33 + r];
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

inline void cut(Prod& g, int bm, int bn, int bk, int slices) {
    g.tiles_n = (g.N + bn - 1) / bn;
    g.tiles = (g.M + bm - 1) / bm * g.tiles_n;
    g.total = g.tiles * slices;
    const int slabs = (g.K + bk - 1) / bk;
    g.slabs = slabs / slices;
    g.slabs_rem = slabs % slices;
}

template <typename T, bool TR, int BM, int BN, int OCC>
void launch_tiles(Prod g, int slices, bool direct, hipStream_t st) {
    // slabs of 64 k; 32 where a slab of 192 x 192 passes through registers, of which 64 would need more than there are
    auto go = [&](auto bk, auto tag) {
        constexpr int BK = decltype(bk)::value;
        constexpr bool DIRECT = decltype(tag)::value;
        cut(g, BM, BN, BK, slices);
        const unsigned grid = (unsigned)((g.total + 7) / 8 * 8);
        half_gemm<T, TR, DIRECT, BM, BN, BK, DIRECT ? OCC : 2><<<grid, 256, 0, st>>>(g);
    };
    if (direct) go(std::integral_constant<int, 64>{}, std::true_type{});
    else go(std::integral_constant<int, BM * BN <= 128 * 192 ? 64 : 32>{}, std::false_type{});
}

inline int64_t tiles_of(int64_t M, int64_t N, int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

// Which kernel a product of M x N results takes.  0: small_gemm, up to 512 tiles of 32 x 32 (512 x 512 x 512 5.0 us against 7.9;
// 2048 x 512 x 512 12.1 against 7.9), up to 64 where rows start off 16-byte borders, whose fragments cost more loads (512 x 800 x
// 513 16.8 against 9.7).  Above, the least of start + share of the chip per 256 tiles, fitted to K = 800 (bf16, GELU, us; the
// times at 4096, 8192, 16384 and 74750 rows of 900); the small ones cost 3.6 and 5.4 where slabs pass through registers (7850 x
// 800 x 513: 27.0 us in 64 x 128 tiles, 23.1 in 128 x 128):
//   1  64 x 64     6 + 2.85, at least 11      18.9   30.6   52.2   210
//   2  64 x 128    6 + 4.6,  at least 13      16.7   27.3   47.7   182
//   3  128 x 128   8 + 8.0,  at least 18      20.8   25.5   40.8   155
//   4  128 x 192   8 + 12,   at least 20      23.1   28.9   39.9   142
// K is not in the rule.  Against all four at K = 64, 65, 333, 512, 513, 800, 801, 4096 and N = 300, 512, 900 its choice is 2 % behind
// the best in the median and 28 % at most (8192 x 65 -> 900: 18.2 against 14.2).
inline int choose_tiles(int64_t M, int64_t N, int64_t K, bool direct) {
    if (K < 8 && !direct) return 0;                                           // no 8 elements in a row to load at once
    if (tiles_of(M, N, 32, 32) <= (direct ? 512 : 64)) return 0;
    static const struct { int bm, bn; double start, per, odd, least; } kind[4] = {
        {64, 64, 6, 2.85, 3.6, 11}, {64, 128, 6, 4.6, 5.4, 13}, {128, 128, 8, 8, 8, 18}, {128, 192, 8, 12, 12, 20}};
    int best = 0;
    double least = 0;
    for (int v = 0; v < 4; ++v) {
        const double t = kind[v].start + (direct ? kind[v].per : kind[v].odd) / 256 * (double)tiles_of(M, N, kind[v].bm, kind[v].bn);
        const double c = t > kind[v].least ? t : kind[v].least;
        if (v == 0 || c < least) { best = v; least = c; }
    }
    return best + 1;
}

template <typename T>
void launch_product(Prod g, bool direct, hipStream_t st) {
    const int v = choose_tiles(g.M, g.N, g.K, direct);
    if (v == 0) {
        g.tiles_n = (g.N + 31) / 32;
        small_gemm<T><<<(unsigned)tiles_of(g.M, g.N, 32, 32), 256, 0, st>>>(g);
    } else if (v == 1) launch_tiles<T, false, 64, 64, 4>(g, 1, direct, st);
    else if (v == 2) launch_tiles<T, false, 64, 128, 4>(g, 1, direct, st);
    else if (v == 3) launch_tiles<T, false, 128, 128, 4>(g, 1, direct, st);
    else launch_tiles<T, false, 128, 192, 3>(g, 1, direct, st);
}

// dW's tiles and the slices of its contraction over R rows (bf16, us, with the launch that adds the slices up).
//   from 8e9 products on, 192 x 192 tiles in one resident round of two workgroups a CU: 900 x 800 over 74750 rows 133 (64 x 64:
//   237), over 16384 rows 44 (53), 512 x 512 over 74750 rows 56 (60)
//   below, 64 x 64 tiles in s slices: a slice's slabs cost about 0.5 each, and s partial tiles are written and read at 4 TB/s, so
//   s = sqrt(slabs * 250000 / (P Q)): 512 x 512 over 16384 rows 21 in 16 slices (192 x 192: 28), over 2048 rows 10 in 6 (16.6),
//   900 x 800 over 4096 rows 21 in 4 (25)
struct DwPlan { bool large; int slices; };
inline DwPlan dw_plan(int64_t R, int64_t P, int64_t Q) {
    DwPlan p;
    p.large = (double)R * (double)P * (double)Q >= 8e9 && tiles_of(P, Q, 192, 192) >= 6;
    const int64_t slabs = (R + 63) / 64;
    int64_t s = p.large ? 512 / tiles_of(P, Q, 192, 192) : (int64_t)(sqrt((double)slabs * 250000.0 / ((double)P * (double)Q)) + 0.5);
    s = s > slabs ? slabs : s;
    p.slices = (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
    return p;
}

struct BwdPlan {
    int log2_lanes, col_tiles, rows_wg, row_wgs;
    DwPlan dw;
    int64_t lddz;
    int64_t off_wt, off_x8, off_part, off_ws, bytes;
};

BwdPlan bwd_plan(int64_t M, int64_t N, int64_t K) {
    BwdPlan p;
    const int64_t groups = (N + 7) / 8;
    p.log2_lanes = 0;
    while (p.log2_lanes < 8 && (int64_t(1) << p.log2_lanes) < groups) ++p.log2_lanes;
    p.col_tiles = (int)((groups + (1 << p.log2_lanes) - 1) >> p.log2_lanes);
    const int slots = 256 >> p.log2_lanes;
    // about 1024 workgroups, at least 4 rows for a thread
    int64_t rows = (M * p.col_tiles + 1023) / 1024;
    rows = (rows + 4 * slots - 1) / (4 * slots) * (4 * slots);
    p.rows_wg = (int)rows;
    p.row_wgs = (int)((M + rows - 1) / rows);
    p.dw = dw_plan(M, N, K);
    p.lddz = (N + 63) / 64 * 64;
    auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    int64_t at = up(M * p.lddz * 2);
    p.off_wt = at;
    at += up(K * p.lddz * 2);
    p.off_x8 = at;
    at += K < 8 ? up(M * 16) : 0;
    p.off_part = at;
    at += up((int64_t)p.row_wgs * N * 4);
    p.off_ws = at;
    at += up((int64_t)p.dw.slices * N * K * 4);
    p.bytes = at;
    return p;
}

bool known_act(int a) { return a == HD_ACT_IDENTITY || a == HD_ACT_RELU || a == HD_ACT_GELU; }

#define HD_LINEAR_SHAPE(fn)                                                                                                     \
    HD_REQUIRE(dtype == HD_DT_BF16 || dtype == HD_DT_F16, fn ": element type bf16 or fp16, not %d", dtype);                      \
    HD_REQUIRE(known_act(act), fn ": activation identity, relu or gelu, not %d", act);                                          \
    HD_REQUIRE(M >= 0 && M < (1LL << 29) && N >= 1 && N < (1LL << 22) && K >= 1 && K < (1LL << 22), fn ": bad shape");             \
    HD_REQUIRE(ldx >= K && ldw >= K, fn ": row pitch below the width")

template <typename T>
int linear_fwd(const Prod& g, bool direct, hipStream_t s) {
    launch_product<T>(g, direct, s);
    return check_launch("hd_linear_act_fwd");
}

template <typename T>
int linear_bwd(const T* g, int64_t ldg, const f16* z, const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t M, int64_t N, int64_t K,
               int act, const T* dx_add, int64_t ld_add, T* dx, T* dw, T* db, const BwdPlan& p, unsigned char* ws, hipStream_t s) {
    const T* dz = g;
    long long lddz = ldg;
    T* wt = (T*)(ws + p.off_wt);
    float* part = db ? (float*)(ws + p.off_part) : nullptr;
    // dz itself is written unless it is g and g's rows can be staged as they are
    const bool copy = (dx || dw) && (act != HD_ACT_IDENTITY || !direct_ok(g, ldg, N, M));
    const int dz_wgs = copy || db ? p.row_wgs * p.col_tiles : 0;
    const int64_t wt_wgs = dx ? ((N + 31) / 32) * ((K + 31) / 32) : 0;
    T* x8 = dw && K < 8 ? (T*)(ws + p.off_x8) : nullptr;
    const int64_t x8_wgs = x8 ? (M + 255) / 256 : 0;
    if (dz_wgs + wt_wgs + x8_wgs)
        act_bwd_k<T><<<(unsigned)(dz_wgs + wt_wgs + x8_wgs), 256, 0, s>>>(g, ldg, z, (int)M, (int)N, act, p.log2_lanes, p.rows_wg, p.col_tiles, dz_wgs,
                                                                copy ? (T*)ws : nullptr, p.lddz, part, w, ldw, (int)K, wt, (int)wt_wgs, x, ldx, x8);
    if (copy) { dz = (const T*)ws; lddz = p.lddz; }
    Prod q = {}, v = {};
    q.act = HD_ACT_IDENTITY;
    q.A = dz; q.lda = lddz;
    v = q;
    // dx: (M, K) = dz (M, N) . W^T (K, N), zeros up to whole chunks;  dW: (N, K) = dz^T (N, M) . x (M, K)
    q.B = wt; q.ldb = p.lddz; q.M = (int)M; q.N = (int)K; q.K = (int)((N + 7) / 8 * 8); q.C = dx; q.resid = dx_add; q.ldr = ld_add;
    v.B = x8 ? x8 : x; v.ldb = x8 ? 8 : ldx; v.M = (int)N; v.N = (int)K; v.K = (int)M; v.C = ws + p.off_ws;
    const bool direct = x8 || direct_ok(x, ldx, K, M);
    if (dx && dw && !p.dw.large && choose_tiles(q.M, q.N, q.K, true) == 0) {
        const int dx_wgs = (int)tiles_of(M, K, 32, 32);
        q.tiles_n = (q.N + 31) / 32;
        cut(v, 64, 64, 64, p.dw.slices);
        if (direct) small_pair<T, true><<<(unsigned)(dx_wgs + v.total), 256, 0, s>>>(q, v, dx_wgs);
        else small_pair<T, false><<<(unsigned)(dx_wgs + v.total), 256, 0, s>>>(q, v, dx_wgs);
    } else {
        if (dx) launch_product<T>(q, true, s);
        if (dw && p.dw.large) launch_tiles<T, true, 192, 192, 2>(v, p.dw.slices, direct, s);
        else if (dw) launch_tiles<T, true, 64, 64, 4>(v, p.dw.slices, direct, s);
    }
    if (dw || db) {
        const int64_t count = dw ? N * K : 0;
        const int w_wgs = (int)((count + 1023) / 1024), b_wgs = db ? (int)((N + 15) / 16) : 0;
        half_reduce_k<T><<<(unsigned)(w_wgs + b_wgs), 256, 0, s>>>((const float*)(ws + p.off_ws), p.dw.slices, count, dw, w_wgs, part,
                                                                   p.row_wgs, (int)N, db);
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
    const bool direct = direct_ok(x, ldx, K, M) && direct_ok(w, ldw, K, N);
    const int64_t tile = K < 8 && !direct ? 32 : 64;                          // small_gemm's tiles, whatever their number
    HD_REQUIRE(tiles_of(M, N, tile, tile) < (1LL << 24) - 8, "hd_linear_act_fwd: too many tiles");   // a grid holds 2^32 threads
    Prod g = {};
    g.A = x; g.lda = ldx; g.B = w; g.ldb = ldw; g.M = (int)M; g.N = (int)N; g.K = (int)K;
    g.C = y; g.bias = bias; g.resid = resid; g.ldr = ldr; g.z = z; g.act = act;
    // a z beside which nothing stays in the 256 MB behind the L2s until the backward pass reads it: 74750 x 900 183 against 200 us
    g.z_past = M * N >= (1LL << 25);
    return dtype == HD_DT_BF16 ? linear_fwd<bf16>(g, direct, (hipStream_t)st) : linear_fwd<f16>(g, direct, (hipStream_t)st);
}

extern "C" int64_t hd_linear_act_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int act) {
    if (M < 0 || N < 1 || K < 1 || M >= (1LL << 29) || N >= (1LL << 22) || K >= (1LL << 22) || !known_act(act)) return 0;
    return bwd_plan(M, N, K).bytes;
}

extern "C" int hd_linear_act_bwd(const void* g, int64_t ldg, const void* z, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                 int dtype, int64_t M, int64_t N, int64_t K, int act, const void* dx_add, int64_t ld_add, void* dx,
                                 void* dw, void* db, void* workspace, int64_t workspace_bytes, void* st) {
    HD_LINEAR_SHAPE("hd_linear_act_bwd");
    HD_REQUIRE(ldg >= N, "hd_linear_act_bwd: row pitch below the width");
    HD_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0, "hd_linear_act_bwd: null or misaligned workspace");
    HD_REQUIRE(!dx_add || (dx && ld_add >= 0), "hd_linear_act_bwd: dx_add without dx, or a negative pitch");
    HD_REQUIRE(M == 0 || (g && (z || act == HD_ACT_IDENTITY)), "hd_linear_act_bwd: null pointer");
    HD_REQUIRE(!(dx && M > 0) || w, "hd_linear_act_bwd: dx needs w");
    HD_REQUIRE(!(dw && M > 0) || x, "hd_linear_act_bwd: dw needs x");
    HD_REQUIRE((((uintptr_t)g | (uintptr_t)z | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db | (uintptr_t)dx_add) & 1) == 0,
               "hd_linear_act_bwd: pointer not aligned to the element");
    HD_REQUIRE(M > 0, "hd_linear_act_bwd: no rows (the gradients are zeros; fill them)");
    const BwdPlan p = bwd_plan(M, N, K);
    HD_REQUIRE(workspace_bytes >= p.bytes, "hd_linear_act_bwd: workspace of %lld bytes required, got %lld", (long long)p.bytes,
               (long long)workspace_bytes);
    HD_REQUIRE(tiles_of(M, K, 64, 64) < (1LL << 24) - 8 && tiles_of(N, K, 32, 32) < (1LL << 23),
               "hd_linear_act_bwd: too many tiles");
    unsigned char* ws = (unsigned char*)workspace;
    hipStream_t s = (hipStream_t)st;
    if (dtype == HD_DT_BF16)
        return linear_bwd<bf16>((const bf16*)g, ldg, (const f16*)z, (const bf16*)x, ldx, (const bf16*)w, ldw, M, N, K, act, (const bf16*)dx_add, ld_add, (bf16*)dx,
                                (bf16*)dw, (bf16*)db, p, ws, s);
    return linear_bwd<f16>((const f16*)g, ldg, (const f16*)z, (const f16*)x, ldx, (const f16*)w, ldw, M, N, K, act, (const f16*)dx_add,
                           ld_add, (f16*)dx, (f16*)dw, (f16*)db, p, ws, s);
}
