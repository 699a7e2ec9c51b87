// AdamW (decoupled weight decay) over many parameter tensors in one launch, moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32, every operation rounded by itself (the build contracts nothing), so that a restatement in elementwise fp32
// operations gives the same bits.  The reference trains with optim.Adam (diff.py:107, diff_graphset.py:66); its
// optimizers/ package offers no decay and no reduced state.
//
// 8-bit moments: a tensor is cut into blocks of 256 elements (its last one may be shorter); a block holds m and
// s = sqrt(v) as e4m3 codes with one fp32 scale each, max|.| / 448.  The root halves the exponent range, so e4m3's 2^17.8
// covers 2^35 of v.  m rounds to nearest (off by 2^-4 relative at most, forgotten at 1 - b1 per step).  s may not: a step
// changes v by at most 1 - b2 = 1e-3 of itself downwards, s by half of that, far below half a code (2^-4), so nearest would
// never let v decay.  The bits that a code drops are compared with the Weyl sequence frac(i * 2654435761 / 2^32 + t *
// 1779033703 / 2^32) of element index and step: equidistributed over t for every element, hence unbiased over steps, and
// the same on every run.  A positive s never becomes code 0 (the quotient m / s would explode).  A block that meets a
// non-finite moment gets the scale NaN: the damage shows in the next step instead of being rounded away.
//
// Bound by HBM: one pass over p, g and the state.  8 consecutive elements a lane (16-byte loads of 16-bit data, 8-byte
// loads of codes), a block = 32 lanes, whose maxima meet in five lane exchanges; no LDS, no second pass.
// 102 M bf16 parameters with fp32 masters and 8-bit moments: 301 us, 5.5 TB/s; 6.4 M with 32-bit moments: 32 us, 5.5 TB/s.
#include "hd_common.cuh"
#include "hd_half.cuh"
#include "../../include/hypdiff.h"

using namespace hd;

namespace {

constexpr int kBlockElems = 256;                    // elements of one scale
constexpr int kPer = 8;                             // consecutive elements of a lane
constexpr int kWg = 256;                            // threads
constexpr int kWgElems = kWg * kPer;                // 8 blocks a workgroup
constexpr int kMaxJobs = 88;                        // 40 bytes each: the argument block stays below 4 KB

struct Jobs {
    int n;
    void* p[kMaxJobs];
    const void* g[kMaxJobs];
    long long first[kMaxJobs];                      // first element in the flat state, a multiple of kBlockElems
    long long count[kMaxJobs];
    unsigned wg0[kMaxJobs];                         // first workgroup of the job
    int row[kMaxJobs];                              // row of the step table
};

struct Hyper {
    float b1, w1, b2, w2, eps, decay, step_size, r2;   // w = 1 - b; r2 = 1 / sqrt(1 - b2^t)
    unsigned t;
};

// {t, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)} of a tensor, on the device: a captured launch replays with the right corrections
__global__ void adamw_tick(const Jobs jobs, double* __restrict__ steps, double lr, double beta1, double beta2) {
    const int k = blockIdx.x * blockDim.x + threadIdx.x;
    if (k >= jobs.n) return;
    double* s = steps + 3 * (long long)jobs.row[k];
    const double t = s[0] + 1.0;
    s[0] = t;
    s[1] = lr / (1.0 - pow(beta1, t));
    s[2] = 1.0 / sqrt(1.0 - pow(beta2, t));
}

// maximum of the 32 lanes that share a block, as unsigned bit patterns of non-negative floats (a NaN is the largest)
template <int CTRL>
__device__ __forceinline__ unsigned max_dpp(unsigned v) {
    const unsigned w = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
    return v > w ? v : w;
}
__device__ __forceinline__ unsigned max32(unsigned v) {
    v = max_dpp<0xB1>(v);                           // lane ^ 1
    v = max_dpp<0x4E>(v);                           // lane ^ 2
    v = max_dpp<0x141>(v);                          // mirror inside 8
    v = max_dpp<0x140>(v);                          // mirror inside 16
    const unsigned w = (unsigned)__builtin_amdgcn_ds_swizzle((int)v, 0x401F);   // lane ^ 16
    return v > w ? v : w;
}

__device__ __forceinline__ void block_scale(unsigned amax_bits, float& scale, float& inv) {
    const float amax = __builtin_bit_cast(float, amax_bits);
    scale = fmaxf(amax, 0x1p-100f) * (1.0f / 448.0f);
    inv = 1.0f / scale;
    if (amax_bits == 0) { scale = 0.f; inv = 0.f; }
    if (amax_bits >= 0x7f800000u) scale = __builtin_bit_cast(float, 0x7fc00000u);
}

// e4m3 code of s * inv >= 0, rounded by the Weyl sequence: bias 127 -> 7, 23 -> 3 mantissa bits
__device__ __forceinline__ unsigned root_code(float s, float inv, unsigned i, unsigned t) {
    const float y = s * inv;
    const unsigned d = (i * 2654435761u + t * 1779033703u) >> 12;           // the 20 bits to compare the dropped ones with
    int code;
    if (y < 0x1p-6f) code = (int)floorf(y * 512.0f + (float)d * 0x1p-20f);     // below the smallest normal: steps of 2^-9
    else code = (int)((__builtin_bit_cast(unsigned, y) + d) >> 20) - 960;
    code = code < 126 ? code : 126;                                            // 448 is the largest
    code = code > 1 ? code : 1;
    return s > 0.f ? (unsigned)code : 0u;
}

__device__ __forceinline__ void decode4(unsigned c, float scale, float* v) {
    v[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * scale;
    v[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1) * scale;
    v[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2) * scale;
    v[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3) * scale;
}

// The state's pointers, already at the segment's first element, and the tensor's
template <typename T> struct Lane {
    T* p;
    const T* g;
    unsigned char *m, *v;
    float *ms, *vs, *master;
};

// One lane's 8 elements from e0 on.  FULL: all lanes of the wavefront are inside the tensor; otherwise element by element up
// to `live`, zeros behind it (a started block's padding is rewritten with zeros, lanes behind the last block write nothing).
template <typename T, int BITS, bool MASTER, bool FULL>
__device__ __forceinline__ void adamw_lane(const Lane<T>& a, const Hyper& h, long long e0, int live, bool in_state) {
    float pv[kPer], gv[kPer], m[kPer], v[kPer], s[kPer];
    const long long es = FULL || in_state ? e0 : 0;                            // a readable place of the state
    if constexpr (FULL) {
        const Pack<T, kPer> x = load_pack<T, kPer>(a.g + e0);
#pragma unroll
        for (int e = 0; e < kPer; ++e) gv[e] = (float)x.v[e];
        if constexpr (!MASTER) {
            const Pack<T, kPer> y = load_pack<T, kPer>(a.p + e0);
#pragma unroll
            for (int e = 0; e < kPer; ++e) pv[e] = (float)y.v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            gv[e] = e < live ? (float)a.g[e0 + e] : 0.f;
            if constexpr (!MASTER) pv[e] = e < live ? (float)a.p[e0 + e] : 0.f;
        }
    }
    if constexpr (MASTER) {
        const Pack<float, kPer> y = load_pack<float, kPer>(a.master + es);
#pragma unroll
        for (int e = 0; e < kPer; ++e) pv[e] = y.v[e];
    }
    if constexpr (BITS == 32) {
        const Pack<float, kPer> x = load_pack<float, kPer>((const float*)a.m + es), y = load_pack<float, kPer>((const float*)a.v + es);
#pragma unroll
        for (int e = 0; e < kPer; ++e) { m[e] = x.v[e]; v[e] = y.v[e]; }
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(a.m + es), y = *reinterpret_cast<const uint2*>(a.v + es);
        const float sm = a.ms[es / kBlockElems], sv = a.vs[es / kBlockElems];
        decode4(x.x, sm, m);
        decode4(x.y, sm, m + 4);
        decode4(y.x, sv, v);
        decode4(y.y, sv, v + 4);
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[e] = v[e] * v[e];
    }
    unsigned am = 0, as = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        m[e] = m[e] * h.b1 + gv[e] * h.w1;
        v[e] = v[e] * h.b2 + (gv[e] * gv[e]) * h.w2;
        s[e] = sqrtf(v[e]);
        pv[e] = pv[e] * h.decay - (m[e] / (s[e] * h.r2 + h.eps)) * h.step_size;
        if (!FULL && e >= live) { m[e] = 0.f; v[e] = 0.f; s[e] = 0.f; pv[e] = 0.f; }
        if constexpr (BITS == 8) {
            const unsigned bm = __builtin_bit_cast(unsigned, m[e]) & 0x7fffffffu, bs = __builtin_bit_cast(unsigned, s[e]) & 0x7fffffffu;
            am = am > bm ? am : bm;
            as = as > bs ? as : bs;
        }
    }
    if constexpr (FULL) {
        Pack<T, kPer> o;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o.v[e] = (T)pv[e];
        store_pack<T, kPer>(a.p + e0, o);
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (e < live) a.p[e0 + e] = (T)pv[e];
    }
    float sm, im, ss, is;
    if constexpr (BITS == 8) {                                                 // every lane of the wavefront takes part
        block_scale(max32(am), sm, im);
        block_scale(max32(as), ss, is);
    }
    if (!FULL && !in_state) return;
    if constexpr (MASTER) {
        Pack<float, kPer> o;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o.v[e] = pv[e];
        store_pack<float, kPer>(a.master + e0, o);
    }
    if constexpr (BITS == 32) {
        Pack<float, kPer> x, y;
#pragma unroll
        for (int e = 0; e < kPer; ++e) { x.v[e] = m[e]; y.v[e] = v[e]; }
        store_pack<float, kPer>((float*)a.m + e0, x);
        store_pack<float, kPer>((float*)a.v + e0, y);
    } else {
        unsigned cm[2], cs[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const unsigned x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[4 * q] * im, m[4 * q + 1] * im, 0, false);
            const unsigned y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(m[4 * q + 2] * im, m[4 * q + 3] * im, 0, false);
            cm[q] = (x & 0xffffu) | (y << 16);
            cs[q] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                cs[q] |= root_code(s[4 * q + e], is, (unsigned)(e0 + 4 * q + e), h.t) << (8 * e);
        }
        *reinterpret_cast<uint2*>(a.m + e0) = make_uint2(cm[0], cm[1]);
        *reinterpret_cast<uint2*>(a.v + e0) = make_uint2(cs[0], cs[1]);
        if ((threadIdx.x & 31) == 0) {
            a.ms[e0 / kBlockElems] = sm;
            a.vs[e0 / kBlockElems] = ss;
        }
    }
}

template <typename T, int BITS, bool MASTER>
__global__ __launch_bounds__(kWg) void adamw_multi(const Jobs jobs, Hyper h, unsigned char* m_flat, unsigned char* v_flat,
                                                   float* m_scale, float* v_scale, float* master, double* steps, int device_count) {
    int lo = 0, hi = jobs.n - 1;                                               // the last job that starts at or before this workgroup
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (jobs.wg0[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    if (device_count) {
        const double* s = steps + 3 * (long long)jobs.row[lo];
        h.t = (unsigned)(unsigned long long)s[0];
        h.step_size = (float)s[1];
        h.r2 = (float)s[2];
    } else if (steps && blockIdx.x == jobs.wg0[lo] && threadIdx.x == 0) {
        steps[3 * (long long)jobs.row[lo]] = (double)h.t;                      // the device's count follows the host's
    }
    const long long count = jobs.count[lo], first = jobs.first[lo];
    Lane<T> a;
    a.p = (T*)jobs.p[lo];
    a.g = (const T*)jobs.g[lo];
    a.m = m_flat + first * (BITS / 8);
    a.v = v_flat + first * (BITS / 8);
    a.ms = m_scale + first / kBlockElems;
    a.vs = v_scale + first / kBlockElems;
    a.master = master + first;
    const long long w0 = (long long)(blockIdx.x - jobs.wg0[lo]) * kWgElems + (threadIdx.x >> 6) * (64 * kPer);   // the wavefront's
    const long long e0 = w0 + (threadIdx.x & 63) * kPer;
    if (w0 + 64 * kPer <= count) {
        adamw_lane<T, BITS, MASTER, true>(a, h, e0, kPer, true);
    } else if (w0 < count) {
        const int live = e0 >= count ? 0 : (count - e0 < kPer ? (int)(count - e0) : kPer);
        adamw_lane<T, BITS, MASTER, false>(a, h, e0, live, e0 < (count + kBlockElems - 1) / kBlockElems * kBlockElems);
    }
}

template <typename T>
void launch(unsigned wgs, hipStream_t st, const Jobs& j, const Hyper& h, int bits, unsigned char* m, unsigned char* v, float* ms, float* vs, float* master,
            double* steps, int device_count) {
    constexpr bool kHalf = sizeof(T) == 2;                                     // an fp32 parameter has no master
    if (bits == 32) {
        if (kHalf && master) adamw_multi<T, 32, kHalf><<<wgs, kWg, 0, st>>>(j, h, m, v, ms, vs, master, steps, device_count);
        else adamw_multi<T, 32, false><<<wgs, kWg, 0, st>>>(j, h, m, v, ms, vs, master, steps, device_count);
    } else {
        if (kHalf && master) adamw_multi<T, 8, kHalf><<<wgs, kWg, 0, st>>>(j, h, m, v, ms, vs, master, steps, device_count);
        else adamw_multi<T, 8, false><<<wgs, kWg, 0, st>>>(j, h, m, v, ms, vs, master, steps, device_count);
    }
}

}  // namespace

extern "C" int64_t hd_adamw_max_jobs(void) { return kMaxJobs; }

extern "C" int hd_adamw_step(const hd_adamw_job* jobs, int n_jobs, int dtype, int state_bits, void* exp_avg, void* exp_avg_sq,
                             void* exp_avg_scale, void* exp_avg_sq_scale, void* master, int64_t state_elems, double lr,
                             double beta1, double beta2, double eps, double weight_decay, int64_t step, void* step_table,
                             int64_t step_rows, void* st) {
    HD_REQUIRE(n_jobs >= 0 && n_jobs <= kMaxJobs && (jobs || n_jobs == 0), "hd_adamw_step: between 0 and %d jobs per call", kMaxJobs);
    HD_REQUIRE(dtype == HD_DT_F32 || dtype == HD_DT_BF16 || dtype == HD_DT_F16, "hd_adamw_step: unknown element type %d", dtype);
    HD_REQUIRE(state_bits == 32 || state_bits == 8, "hd_adamw_step: moments in 32 or 8 bits, not %d", state_bits);
    HD_REQUIRE(!(master && dtype == HD_DT_F32), "hd_adamw_step: an fp32 parameter is its own master");
    HD_REQUIRE(lr >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && weight_decay >= 0.0,
               "hd_adamw_step: bad hyper-parameters");
    HD_REQUIRE(step >= 0 && (step >= 1 || step_table), "hd_adamw_step: a step count from 1, or a step table");
    HD_REQUIRE(state_elems >= 0 && state_elems % kBlockElems == 0, "hd_adamw_step: the flat state holds whole blocks of %d", kBlockElems);
    Jobs j;
    j.n = 0;
    uint64_t wgs = 0;
    for (int i = 0; i < n_jobs; ++i) {
        if (jobs[i].count == 0) continue;
        HD_REQUIRE(jobs[i].param && jobs[i].grad && jobs[i].count > 0, "hd_adamw_step: job %d: null pointer or negative count", i);
        HD_REQUIRE((uintptr_t)jobs[i].param % dt_size(dtype) == 0 && (uintptr_t)jobs[i].grad % dt_size(dtype) == 0,
                   "hd_adamw_step: job %d: pointer not aligned to the element", i);
        HD_REQUIRE(jobs[i].first >= 0 && jobs[i].first % kBlockElems == 0 && jobs[i].count <= state_elems &&
                       jobs[i].first <= state_elems - (jobs[i].count + kBlockElems - 1) / kBlockElems * kBlockElems,
                   "hd_adamw_step: job %d: segment outside the flat state or not on a block's border", i);
        HD_REQUIRE(!step_table || (jobs[i].row >= 0 && jobs[i].row < step_rows), "hd_adamw_step: job %d: row outside the step table", i);
        const int k = j.n++;
        j.p[k] = jobs[i].param;
        j.g[k] = jobs[i].grad;
        j.first[k] = jobs[i].first;
        j.count[k] = jobs[i].count;
        j.row[k] = (int)jobs[i].row;
        j.wg0[k] = (unsigned)wgs;
        wgs += (uint64_t)(jobs[i].count + kWgElems - 1) / kWgElems;
        HD_REQUIRE(wgs < (1ULL << 24), "hd_adamw_step: too many elements in one call");      // a grid holds 2^32 threads
    }
    if (j.n == 0) return HD_OK;
    HD_REQUIRE(exp_avg && exp_avg_sq && (state_bits == 32 || (exp_avg_scale && exp_avg_sq_scale)), "hd_adamw_step: null state");
    HD_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)master) & 15) == 0, "hd_adamw_step: state not 16-byte aligned");
    const double t = step >= 1 ? (double)step : 1.0;
    Hyper h;
    h.b1 = (float)beta1;
    h.w1 = (float)(1.0 - beta1);
    h.b2 = (float)beta2;
    h.w2 = (float)(1.0 - beta2);
    h.eps = (float)eps;
    h.decay = (float)(1.0 - lr * weight_decay);
    h.step_size = (float)(lr / (1.0 - pow(beta1, t)));
    h.r2 = (float)(1.0 / sqrt(1.0 - pow(beta2, t)));
    h.t = (unsigned)step;
    hipStream_t s = (hipStream_t)st;
    const int device_count = step == 0;
    if (device_count) adamw_tick<<<(j.n + 63) / 64, 64, 0, s>>>(j, (double*)step_table, lr, beta1, beta2);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        launch<T>((unsigned)wgs, s, j, h, state_bits, (unsigned char*)exp_avg, (unsigned char*)exp_avg_sq, (float*)exp_avg_scale,
                  (float*)exp_avg_sq_scale, (float*)master, (double*)step_table, device_count);
    };
    if (dtype == HD_DT_F32) go(float{});
    else if (dtype == HD_DT_BF16) go(bf16{});
    else go(f16{});
    return check_launch("hd_adamw_step");
}
