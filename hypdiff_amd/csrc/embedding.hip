// Embedding lookup  out[r] = add[r] + scale * table[idx[r]]  and its table gradient  dT[v] = scale * sum_{idx[r] = v} g[r],
// in fp32, bf16 or fp16 (the sums in fp32, rounded once).  The time embedding of the graph-level denoiser (ddpm.py:36-41)
// is such a lookup; hd_embedding_add / hd_embedding_grad_f32 are its fp32 form for a caller that sorts by itself.
//
// The gradient is a segment sum over the rows of g in the order of a stable sort by token: every table row is written once,
// by one lane per column, so there are no atomics on floats, the sums run in ascending row order inside fixed chunks, and
// a repeated call gives the same bits.
//   sort    key = token (the padding token and tokens outside the table become T, behind all others), value = row.  Up to
//           512 rows: one workgroup, bitonic on (key, row) in LDS, three launches fewer (the whole gradient of 200 rows 15.0 us,
//           by radix 16.3; of 512 17.8 and 16.7 beside the host's part of the launches; of 4096 47 and 21).
//           More: least-significant-digit radix passes of at most 8 bits; a workgroup counts its own digits' places from the
//           counts of all workgroups (at most 256 of them, one read of 256 KB): two launches a pass.  (Counting the next
//           pass's digits in the scatter, by atomics on the counts of the workgroup a row moves to, saved a launch of 3 us
//           and cost 11: the rows of a hot token meet on one counter.)
//   sum     the sorted rows are cut into chunks of P; a lane owns VEC columns, walks a chunk and writes a table row
//           whenever a run ends.  A run that crosses a chunk's border leaves a partial sum there, which the next launch
//           adds up in chunk order: a hot token (18 000 of 75 000 rows) is spread over hundreds of wavefronts.  Further
//           workgroups of the same launch write the zeros of the table rows that no row names.
// A width that is no multiple of VEC: the last lane takes the last VEC columns, some of them a second time, with equal results
// (branches for its short group cost half of the time: loads that wait for each other).
// Bound by HBM: one read of g and one write of the table's gradient (the lookup: one read of the named rows, one write).
// 131072 x 700 bf16 of 50000 tokens: lookup 61 us (6.0 TB/s), sort 20, sum 74 (3.4 TB/s), join 11.  74750 x 512 fp32 of 1000,
// unevenly drawn: lookup 52 (5.9 TB/s), sort 17, sum 44 (3.5 TB/s), join 10; the sum takes 26 where g is still in the caches.
#include <type_traits>
#include "hd_common.cuh"
#include "hd_half.cuh"
#include "../../include/hypdiff.h"

using namespace hd;

namespace {

constexpr int kSmallRows = 512;                     // rows that one workgroup sorts
constexpr int kSmallWg = 256;
constexpr int kSortWg = 1024;
constexpr int kMaxSortWgs = 256;
constexpr int kZeroRows = 64;                       // table rows of one zero-writing workgroup
constexpr int64_t kLookupRows = 1 << 25;            // rows of one lookup launch: a grid holds 2^32 threads

// ---- lookup ---------------------------------------------------------------------------------------------------------------
template <typename T, int VEC, typename I>
__global__ __launch_bounds__(256) void lookup_k(const T* __restrict__ table, long long ldt, const I* __restrict__ idx,
                                                const T* __restrict__ add, long long lda, float scale, long long n_table,
                                                long long rows, int dim, int log2_lanes, T* __restrict__ out) {
    const int lanes = 1 << log2_lanes;                                        // lanes of a row (a power of two up to 64)
    const long long r = (long long)blockIdx.x * (256 >> log2_lanes) + (threadIdx.x >> log2_lanes);
    if (r >= rows) return;
    const long long t = (long long)idx[r];
    const bool inside = t >= 0 && t < n_table;                                // outside the table: a row of NaN
    const T* src = table + (inside ? t : 0) * ldt;
    const T* plus = add ? add + r * lda : nullptr;
    T* dst = out + r * dim;
    constexpr int U = 4;                                                      // chunks in flight
    for (int c0 = (threadIdx.x & (lanes - 1)) * VEC; c0 < dim; c0 += U * lanes * VEC) {
        Pack<T, VEC> a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int c = c0 + u * lanes * VEC;
            c = c + VEC <= dim ? c : dim - VEC;
            a[u] = load_pack<T, VEC>(src + c);
            if (plus) b[u] = load_pack<T, VEC>(plus + c);                     // uniform
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int c = c0 + u * lanes * VEC;
            if (c >= dim) break;
            c = c + VEC <= dim ? c : dim - VEC;
            Pack<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float v = scale * (float)a[u].v[e];
                if (plus) v = (float)b[u].v[e] + v;
                o.v[e] = (T)(inside ? v : __builtin_nanf(""));
            }
            store_pack<T, VEC>(dst + c, o);
        }
    }
}

// ---- sort -----------------------------------------------------------------------------------------------------------------
template <typename I>
__device__ __forceinline__ unsigned key_of(I t, long long padding, unsigned n_table) {
    const long long v = (long long)t;
    return v >= 0 && v < (long long)n_table && v != padding ? (unsigned)v : n_table;
}

template <typename I>
__global__ __launch_bounds__(kSmallWg) void sort_small_k(const I* __restrict__ idx, long long padding, unsigned n_table, int n, int n2,
                                                        unsigned* __restrict__ keys, unsigned* __restrict__ pos) {
    __shared__ unsigned long long s[kSmallRows];
    for (int i = threadIdx.x; i < n2; i += kSmallWg)
        s[i] = i < n ? ((unsigned long long)key_of(idx[i], padding, n_table) << 32) | (unsigned)i : ~0ull;
    __syncthreads();
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < n2 >> 1; i += kSmallWg) {
                const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
                const unsigned long long x = s[a], y = s[b];
                if ((x > y) == ((a & k) == 0)) { s[a] = y; s[b] = x; }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < n; i += kSmallWg) {
        keys[i] = (unsigned)(s[i] >> 32);
        pos[i] = (unsigned)s[i];
    }
}

// digit counts of a pass, [workgroup][256].  FIRST: keys come from idx
template <typename I, bool FIRST>
__global__ __launch_bounds__(kSortWg) void radix_count_k(const I* __restrict__ idx, long long padding, unsigned n_table,
                                                         const unsigned* __restrict__ keys, unsigned n, unsigned per_wg, int shift,
                                                         unsigned mask, unsigned* __restrict__ hist) {
    __shared__ unsigned h[4][256];                                            // four copies: fewer meet on a hot token's counter
    (&h[0][0])[threadIdx.x] = 0;
    __syncthreads();
    const unsigned i0 = blockIdx.x * per_wg, i1 = n - i0 < per_wg ? n : i0 + per_wg;
    for (unsigned i = i0 + threadIdx.x; i < i1; i += kSortWg) {
        unsigned key;
        if constexpr (FIRST) key = key_of(idx[i], padding, n_table);
        else key = keys[i];
        atomicAdd(&h[threadIdx.x & 3][(key >> shift) & mask], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 256) hist[blockIdx.x * 256 + threadIdx.x] = h[0][threadIdx.x] + h[1][threadIdx.x] + h[2][threadIdx.x] + h[3][threadIdx.x];
}

// One stable scatter by the digit (key >> shift) & mask
template <typename I, bool FIRST>
__global__ __launch_bounds__(kSortWg) void radix_scatter_k(const I* __restrict__ idx, long long padding, unsigned n_table,
                                                           const unsigned* __restrict__ keys_in, const unsigned* __restrict__ pos_in,
                                                           unsigned n, unsigned per_wg, int shift, unsigned mask,
                                                           const unsigned* __restrict__ hist, unsigned* __restrict__ keys_out,
                                                           unsigned* __restrict__ pos_out) {
    __shared__ unsigned part_all[4][256], part_before[4][256], place[256], wave_count[16][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, digit = tid & 255, quarter = tid >> 8;
    // where this workgroup's rows of each digit go: all rows of smaller digits, then the earlier workgroups' of this digit
    unsigned all = 0, before = 0;
#pragma unroll 8
    for (unsigned b = quarter; b < gridDim.x; b += 4) {
        const unsigned c = hist[b * 256 + digit];
        all += c;
        before += b < blockIdx.x ? c : 0u;
    }
    part_all[quarter][digit] = all;
    part_before[quarter][digit] = before;
    __syncthreads();
    if (tid < 64) {                                                           // exclusive scan over 256 digits, 4 a lane
        unsigned c[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = tid * 4 + k;
            c[k] = part_all[0][d] + part_all[1][d] + part_all[2][d] + part_all[3][d];
            sum += c[k];
        }
        unsigned run = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned up = (unsigned)__shfl_up((int)run, o);
            if (tid >= o) run += up;
        }
        run -= sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = tid * 4 + k;
            place[d] = run + part_before[0][d] + part_before[1][d] + part_before[2][d] + part_before[3][d];
            run += c[k];
        }
    }
    const unsigned i0 = blockIdx.x * per_wg, i1 = n - i0 < per_wg ? n : i0 + per_wg;
    for (unsigned r = i0; r < i1; r += kSortWg) {                              // rounds of 1024 rows in order
        for (int k = tid; k < 16 * 256; k += kSortWg) (&wave_count[0][0])[k] = 0;
        __syncthreads();                                                      // (also: place is complete / was advanced)
        const unsigned i = r + tid;
        const bool live = i < i1;
        unsigned key = 0, row = i;
        if (live) {
            if constexpr (FIRST) key = key_of(idx[i], padding, n_table);
            else { key = keys_in[i]; row = pos_in[i]; }
        }
        const unsigned d = (key >> shift) & mask;
        // the lanes of this wavefront with the same digit
        unsigned long long same = __ballot(live);
#pragma unroll
        for (int bit = 0; bit < 8; ++bit) {
            const unsigned long long m = __ballot(live && ((d >> bit) & 1));
            same &= (d >> bit) & 1 ? m : ~m;
        }
        const unsigned rank = (unsigned)__popcll(same & ((1ull << lane) - 1));
        if (live && rank == 0) wave_count[wave][d] = (unsigned)__popcll(same);
        __syncthreads();
        if (tid < 256) {                                                      // first place of every wavefront's rows of a digit
            unsigned p = place[tid];
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const unsigned c = wave_count[w][tid];
                wave_count[w][tid] = p;
                p += c;
            }
            place[tid] = p;
        }
        __syncthreads();
        if (live) {
            const unsigned to = wave_count[wave][d] + rank;
            keys_out[to] = key;
            pos_out[to] = row;
        }
        __syncthreads();
    }
}

// ---- sum ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned lower_bound(const unsigned* keys, unsigned n, unsigned v) {
    unsigned lo = 0, hi = n;
    while (lo < hi) {
        const unsigned mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    return lo;
}

template <int VEC>
__device__ __forceinline__ void store_part(float* p, const float (&acc)[VEC]) {
    Pack<float, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = acc[e];
    store_pack<float, VEC>(p, o);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&acc)[VEC], float scale) {
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = (T)(acc[e] * scale);
    store_pack<T, VEC>(p, o);
}

// head[chunk]: the sum of the chunk's rows that continue the run of the chunk before; tail[chunk]: of the run that begins in
// the chunk and goes on in the next.  A lane owns the columns c .. c + VEC - 1 of one chunk.  ONE: a wavefront is in one chunk, so
// that its keys and rows are scalar loads and the ends of runs scalar branches.
template <typename T, int VEC, bool ONE>
__global__ __launch_bounds__(256) void segment_sum_k(const T* __restrict__ g, long long ldg, const unsigned* __restrict__ keys,
                                                     const unsigned* __restrict__ pos, unsigned n, int dim, unsigned n_table,
                                                     float scale, int chunk, int log2_lanes, int tiles, unsigned sum_wgs,
                                                     T* __restrict__ out, float* __restrict__ head, float* __restrict__ tail) {
    if (blockIdx.x >= sum_wgs) {                                              // zeros of the table rows that nothing names
        // a search for every row's first place: walking the keys of 64 rows instead takes one workgroup 90 us where 75 000 rows
        // are one token's
        __shared__ unsigned place[kZeroRows + 1];
        const unsigned t0 = (blockIdx.x - sum_wgs) * kZeroRows;
        const unsigned t1 = n_table - t0 < kZeroRows ? n_table : t0 + kZeroRows;
        if (threadIdx.x <= kZeroRows) place[threadIdx.x] = lower_bound(keys, n, t0 + threadIdx.x);
        __syncthreads();
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const float zero[VEC] = {};
        for (unsigned t = t0 + wave; t < t1; t += 4)
            if (place[t - t0] == place[t - t0 + 1])
                for (int c = lane * VEC; c < dim; c += 64 * VEC)
                    store_row<T, VEC>(out + (long long)t * dim + (c + VEC <= dim ? c : dim - VEC), zero, 1.f);
        return;
    }
    unsigned item = blockIdx.x * (256u >> log2_lanes) + (threadIdx.x >> log2_lanes);
    if constexpr (ONE) item = (unsigned)__builtin_amdgcn_readfirstlane((int)item);
    const unsigned ch = item / (unsigned)tiles;
    int c = ((int)(item - ch * tiles) * (1 << log2_lanes) + (int)(threadIdx.x & ((1 << log2_lanes) - 1))) * VEC;
    const unsigned i0 = ch * chunk;
    if (i0 >= n || c >= dim) return;
    c = c + VEC <= dim ? c : dim - VEC;
    const unsigned i1 = n - i0 < (unsigned)chunk ? n : i0 + chunk;
    const unsigned after = i1 < n ? keys[i1] : ~0u;
    unsigned cur = keys[i0];
    bool cont = i0 > 0 && keys[i0 - 1] == cur;                                // the run began in an earlier chunk
    float acc[VEC] = {};
    constexpr int U = 8;                                                      // rows in flight
    unsigned k[U], p[U];
    auto names = [&](unsigned i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned j = i + u < i1 ? i + u : i1 - 1;
            k[u] = i + u < i1 ? keys[j] : ~0u;
            p[u] = pos[j];
        }
    };
    names(i0);
    for (unsigned i = i0; i < i1; i += U) {
        Pack<T, VEC> x[U];
        unsigned kk[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kk[u] = k[u];
            x[u] = load_pack<T, VEC>(g + (long long)p[u] * ldg + c);
        }
        if (i + U < i1) names(i + U);                                         // on their way while the rows are
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kk[u] == ~0u) break;
            if (kk[u] != cur) {                                               // the run of cur is over
                if (cont) store_part<VEC>(head + (long long)ch * dim + c, acc);
                else if (cur < n_table) store_row<T, VEC>(out + (long long)cur * dim + c, acc, scale);
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
                cur = kk[u];
                cont = false;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += (float)x[u].v[e];
        }
    }
    if (cont) store_part<VEC>(head + (long long)ch * dim + c, acc);
    else if (after == cur) store_part<VEC>(tail + (long long)ch * dim + c, acc);
    else if (cur < n_table) store_row<T, VEC>(out + (long long)cur * dim + c, acc, scale);
}

// Runs that cross chunks: tail of the chunk where the run begins, then the heads up to the chunk where it ends, in order;
// four wavefronts take a quarter of the heads each.  One workgroup per (chunk, 64 VEC columns); chunks without a tail leave at once.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void segment_join_k(const unsigned* __restrict__ keys, unsigned n, int dim, unsigned n_table,
                                                      float scale, int chunk, int tiles, const float* __restrict__ head,
                                                      const float* __restrict__ tail, T* __restrict__ out) {
    __shared__ float red[4][64][VEC];
    __shared__ unsigned last;
    const unsigned ch = blockIdx.x / (unsigned)tiles;
    const unsigned i0 = ch * chunk, i1 = i0 + chunk;                          // the last chunk has no tail: not launched for it
    const unsigned cur = keys[i1 - 1];
    if (cur >= n_table || keys[i1] != cur || (keys[i0] == cur && i0 > 0 && keys[i0 - 1] == cur)) return;
    if (i1 + chunk < n && keys[i1 + chunk] == cur) {                          // it goes on behind the next chunk: where does it end?
        if (threadIdx.x == 0) last = (lower_bound(keys, n, cur + 1) - 1) / (unsigned)chunk;
        __syncthreads();
    } else {
        if (threadIdx.x == 0) last = ch + 1;
        __syncthreads();
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int c = ((int)(blockIdx.x - ch * tiles) * 64 + lane) * VEC;
    const bool live = c < dim;
    c = c + VEC <= dim ? c : dim - VEC;
    const unsigned heads = last - ch, per = (heads + 3) / 4;
    const unsigned a = ch + 1 + wave * per, b = a + per < last + 1 ? a + per : last + 1;
    float acc[VEC] = {};
    auto add = [&](const float* row) {
        const Pack<float, VEC> x = load_pack<float, VEC>(row + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += x.v[e];
    };
    if (wave == 0) add(tail + (long long)ch * dim);
#pragma unroll 8
    for (unsigned k = a; k < b; ++k) add(head + (long long)k * dim);
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[wave][lane][e] = acc[e];
    __syncthreads();
    if (wave == 0 && live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = ((red[0][lane][e] + red[1][lane][e]) + red[2][lane][e]) + red[3][lane][e];
        store_row<T, VEC>(out + (long long)cur * dim + c, acc, scale);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
inline int ceil_log2(int64_t v) {
    int l = 0;
    while ((int64_t(1) << l) < v) ++l;
    return l;
}

// columns of a lane: the widest load (16 bytes at most) that leaves at most a quarter of the lanes without columns
inline int pick_vec(int64_t dim, int most) {
    for (int v = most; v > 1; v >>= 1) {
        const int64_t used = (dim + v - 1) / v, lanes = used > 64 ? (used + 63) / 64 * 64 : int64_t(1) << ceil_log2(used);
        if (4 * used >= 3 * lanes && dim >= v) return v;
    }
    return 1;
}

struct Plan {
    int vec, log2_lanes, tiles, chunk;
    int64_t chunks;
    int passes, width, sort_wgs;
    int64_t per_wg;
    int64_t off_pos, off_keys2, off_pos2, off_hist, off_head, off_tail, bytes;
};

Plan make_plan(int64_t rows, int64_t dim, int64_t n_table, int dt) {
    Plan p;
    p.vec = pick_vec(dim, dt == HD_DT_F32 ? 4 : 8);
    const int64_t used = (dim + p.vec - 1) / p.vec;
    p.log2_lanes = used >= 64 ? 6 : ceil_log2(used);
    p.tiles = (int)((used + (1 << p.log2_lanes) - 1) >> p.log2_lanes);
    // chunks long enough that the partial sums are a small part of the traffic (2 / 64 at the border of every chunk) and
    // short enough that a small batch still fills the chip
    const int64_t lanes_per_row = (int64_t)p.tiles << p.log2_lanes;
    p.chunk = 8;
    while (p.chunk < 64 && rows * lanes_per_row / (2 * p.chunk) >= 2048 * 64) p.chunk *= 2;
    p.chunks = (rows + p.chunk - 1) / p.chunk;
    const int bits = ceil_log2(n_table + 1) > 0 ? ceil_log2(n_table + 1) : 1;     // keys are 0 .. n_table
    p.passes = (bits + 7) / 8;
    p.width = (bits + p.passes - 1) / p.passes;
    int64_t per = (rows + kMaxSortWgs - 1) / kMaxSortWgs;
    per = (per + kSortWg - 1) / kSortWg * kSortWg;
    p.per_wg = per < kSortWg ? kSortWg : per;
    p.sort_wgs = (int)((rows + p.per_wg - 1) / p.per_wg);
    const bool small = rows <= kSmallRows;
    auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    int64_t at = up(rows * 4);                                                   // the sorted keys come first
    p.off_pos = at;
    at += up(rows * 4);
    p.off_keys2 = at;
    at += small ? 0 : up(rows * 4);
    p.off_pos2 = at;
    at += small ? 0 : up(rows * 4);
    p.off_hist = at;
    at += small ? 0 : up((int64_t)p.sort_wgs * 256 * 4);
    p.off_head = at;
    at += up(p.chunks * dim * 4);
    p.off_tail = at;
    at += up(p.chunks * dim * 4);
    p.bytes = at > 256 ? at : 256;
    return p;
}

template <typename I>
void sort_rows(const I* idx, long long padding, unsigned n_table, int64_t rows, const Plan& p, unsigned char* ws, hipStream_t st) {
    unsigned *keys = (unsigned*)ws, *pos = (unsigned*)(ws + p.off_pos);
    if (rows <= kSmallRows) {
        int n2 = 2;
        while (n2 < rows) n2 <<= 1;
        sort_small_k<I><<<1, kSmallWg, 0, st>>>(idx, padding, n_table, (int)rows, n2, keys, pos);
        return;
    }
    unsigned* buf_k[2] = {keys, (unsigned*)(ws + p.off_keys2)};
    unsigned* buf_p[2] = {pos, (unsigned*)(ws + p.off_pos2)};
    unsigned* hist = (unsigned*)(ws + p.off_hist);
    const unsigned mask = (1u << p.width) - 1, n = (unsigned)rows, per = (unsigned)p.per_wg;
    int to = (p.passes - 1) & 1;                                                 // so that the last pass writes buffer 0
    for (int k = 0; k < p.passes; ++k, to ^= 1) {
        const int shift = k * p.width;
        if (k == 0) {
            radix_count_k<I, true><<<p.sort_wgs, kSortWg, 0, st>>>(idx, padding, n_table, nullptr, n, per, shift, mask, hist);
            radix_scatter_k<I, true><<<p.sort_wgs, kSortWg, 0, st>>>(idx, padding, n_table, nullptr, nullptr, n, per, shift, mask, hist,
                                                                     buf_k[to], buf_p[to]);
        } else {
            radix_count_k<I, false><<<p.sort_wgs, kSortWg, 0, st>>>(idx, padding, n_table, buf_k[to ^ 1], n, per, shift, mask, hist);
            radix_scatter_k<I, false><<<p.sort_wgs, kSortWg, 0, st>>>(idx, padding, n_table, buf_k[to ^ 1], buf_p[to ^ 1], n, per, shift,
                                                                      mask, hist, buf_k[to], buf_p[to]);
        }
    }
}

template <typename T, int VEC>
void sum_rows(const T* g, int64_t ldg, int64_t rows, int64_t dim, int64_t n_table, float scale, const Plan& p, unsigned char* ws, T* out,
              hipStream_t st) {
    const unsigned *keys = (const unsigned*)ws, *pos = (const unsigned*)(ws + p.off_pos);
    float *head = (float*)(ws + p.off_head), *tail = (float*)(ws + p.off_tail);
    const int64_t per_wg = 256 >> p.log2_lanes;
    const unsigned sum_wgs = (unsigned)((p.chunks * p.tiles + per_wg - 1) / per_wg);
    const unsigned zero_wgs = (unsigned)((n_table + kZeroRows - 1) / kZeroRows);
    auto go = [&](auto one) {
        segment_sum_k<T, VEC, decltype(one)::value><<<sum_wgs + zero_wgs, 256, 0, st>>>(g, ldg, keys, pos, (unsigned)rows, (int)dim,
                                                                                       (unsigned)n_table, scale, p.chunk, p.log2_lanes,
                                                                                       p.tiles, sum_wgs, out, head, tail);
    };
    if (p.log2_lanes == 6) go(std::true_type{});
    else go(std::false_type{});
    if (p.chunks > 1) {
        auto join = [&](auto vec) {
            constexpr int V = decltype(vec)::value;
            const int tiles = (int)((dim + 64 * V - 1) / (64 * V));
            segment_join_k<T, V><<<(unsigned)((p.chunks - 1) * tiles), 256, 0, st>>>(keys, (unsigned)rows, (int)dim, (unsigned)n_table, scale,
                                                                                     p.chunk, tiles, head, tail, out);
        };
        if (dim >= 4) join(std::integral_constant<int, 4>{});
        else join(std::integral_constant<int, 1>{});
    }
}

template <typename T>
void sum_any(const T* g, int64_t ldg, int64_t rows, int64_t dim, int64_t n_table, float scale, const Plan& p, unsigned char* ws, T* out,
             hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (p.vec == 8) return sum_rows<T, 8>(g, ldg, rows, dim, n_table, scale, p, ws, out, st);
    }
    if (p.vec == 4) return sum_rows<T, 4>(g, ldg, rows, dim, n_table, scale, p, ws, out, st);
    if (p.vec == 2) return sum_rows<T, 2>(g, ldg, rows, dim, n_table, scale, p, ws, out, st);
    return sum_rows<T, 1>(g, ldg, rows, dim, n_table, scale, p, ws, out, st);
}

template <typename T, typename I>
void lookup_any(const T* table, int64_t ldt, const I* idx, const T* add, int64_t lda, float scale, int64_t n_table, int64_t rows,
                int64_t dim, T* out, hipStream_t st) {
    constexpr int MOST = 16 / sizeof(T);
    const int vec = pick_vec(dim, MOST);
    const int64_t used = (dim + vec - 1) / vec;
    const int l2 = used >= 64 ? 6 : ceil_log2(used);
    auto go = [&](auto tag) {
        constexpr int VEC = decltype(tag)::value;
        for (int64_t r = 0; r < rows; r += kLookupRows) {
            const int64_t n = rows - r < kLookupRows ? rows - r : kLookupRows;
            lookup_k<T, VEC, I><<<(unsigned)((n + (256 >> l2) - 1) / (256 >> l2)), 256, 0, st>>>(
                table, ldt, idx + r, add ? add + r * lda : nullptr, lda, scale, n_table, n, (int)dim, l2, out + r * dim);
        }
    };
    if constexpr (MOST == 8) {
        if (vec == 8) return go(std::integral_constant<int, 8>{});
    }
    if (vec == 4) go(std::integral_constant<int, 4>{});
    else if (vec == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
}

bool known_dt(int dt) { return dt == HD_DT_F32 || dt == HD_DT_BF16 || dt == HD_DT_F16; }

}  // namespace

extern "C" int hd_embedding_lookup(const void* table, int64_t ldt, const void* idx, int idx_bits, const void* add, int64_t lda,
                                   double scale, int dtype, int64_t T, int64_t rows, int64_t dim, void* out, void* st) {
    HD_REQUIRE(known_dt(dtype), "hd_embedding_lookup: unknown element type %d", dtype);
    HD_REQUIRE(idx_bits == 32 || idx_bits == 64, "hd_embedding_lookup: indices of 32 or 64 bits, not %d", idx_bits);
    HD_REQUIRE(rows >= 0 && rows < (1LL << 31) && dim >= 1 && dim < (1LL << 30) && T >= 1 && T < (1LL << 31) - 1 && ldt >= 0 && lda >= 0,
               "hd_embedding_lookup: bad shape");
    if (rows == 0) return HD_OK;
    HD_REQUIRE(table && idx && out, "hd_embedding_lookup: null pointer");
    const int es = dt_size(dtype);
    HD_REQUIRE((uintptr_t)table % es == 0 && (uintptr_t)out % es == 0 && (uintptr_t)add % es == 0 && (uintptr_t)idx % (idx_bits / 8) == 0,
               "hd_embedding_lookup: pointer not aligned to the element");
    hipStream_t s = (hipStream_t)st;
    auto go = [&](auto tag) {
        using E = decltype(tag);
        if (idx_bits == 64) lookup_any<E, long long>((const E*)table, ldt, (const long long*)idx, (const E*)add, lda, (float)scale, T, rows, dim, (E*)out, s);
        else lookup_any<E, int>((const E*)table, ldt, (const int*)idx, (const E*)add, lda, (float)scale, T, rows, dim, (E*)out, s);
    };
    if (dtype == HD_DT_F32) go(float{});
    else if (dtype == HD_DT_BF16) go(bf16{});
    else go(f16{});
    return check_launch("hd_embedding_lookup");
}

extern "C" int64_t hd_embedding_sum_workspace_bytes(int64_t rows, int64_t dim, int64_t T, int dtype) {
    if (rows < 0 || dim < 1 || T < 1 || rows >= (1LL << 31) || T >= (1LL << 31) - 1 || dim >= (1LL << 30) || !known_dt(dtype)) return 0;
    return make_plan(rows, dim, T, dtype).bytes;
}

extern "C" int hd_embedding_sum(const void* g, int64_t ldg, const void* idx, int idx_bits, int64_t padding, double scale, int dtype,
                                int64_t T, int64_t rows, int64_t dim, void* out, void* workspace, int64_t workspace_bytes, void* st) {
    HD_REQUIRE(known_dt(dtype), "hd_embedding_sum: unknown element type %d", dtype);
    HD_REQUIRE(idx_bits == 32 || idx_bits == 64, "hd_embedding_sum: indices of 32 or 64 bits, not %d", idx_bits);
    HD_REQUIRE(rows >= 0 && rows < (1LL << 31) && dim >= 1 && dim < (1LL << 30) && T >= 1 && T < (1LL << 31) - 1 && ldg >= 0,
               "hd_embedding_sum: bad shape");
    HD_REQUIRE(out && workspace && (rows == 0 || (g && idx)), "hd_embedding_sum: null pointer");
    const int es = dt_size(dtype);
    HD_REQUIRE((uintptr_t)g % es == 0 && (uintptr_t)out % es == 0 && (uintptr_t)idx % (idx_bits / 8) == 0 && (uintptr_t)workspace % 16 == 0,
               "hd_embedding_sum: misaligned pointer");
    const Plan p = make_plan(rows, dim, T, dtype);
    HD_REQUIRE(workspace_bytes >= p.bytes, "hd_embedding_sum: workspace of %lld bytes required, got %lld", (long long)p.bytes,
               (long long)workspace_bytes);
    HD_REQUIRE(p.chunks * (dim < 4 ? 1 : (dim + 255) / 256) < (1LL << 24) &&
                   ((p.chunks * p.tiles) >> (8 - p.log2_lanes)) + T / kZeroRows < (1LL << 24) - 2,                // a grid holds 2^32 threads
               "hd_embedding_sum: too many workgroups");
    hipStream_t s = (hipStream_t)st;
    unsigned char* ws = (unsigned char*)workspace;
    if (rows > 0) {
        if (idx_bits == 64) sort_rows<long long>((const long long*)idx, padding, (unsigned)T, rows, p, ws, s);
        else sort_rows<int>((const int*)idx, padding, (unsigned)T, rows, p, ws, s);
    }
    auto go = [&](auto tag) {
        using E = decltype(tag);
        sum_any<E>((const E*)g, ldg, rows, dim, T, (float)scale, p, ws, (E*)out, s);
    };
    if (dtype == HD_DT_F32) go(float{});
    else if (dtype == HD_DT_BF16) go(bf16{});
    else go(f16{});
    return check_launch("hd_embedding_sum");
}
