// zs_logprobs.cuh -- log probabilities of given tokens, entropy, log-sum-exp and the
// top alternatives of each row of logits, and their gradient.
//
// With it = inv_temp, m = max x, s = sum_v exp((x_v - m) it):
//   log p_v = (x_v - m) it - ln s         lse = m it + ln s
//   H = -sum_v p_v log p_v = ln s - (sum_v e_v t_v) / s,  t_v = (x_v - m) it, e_v = exp(t_v)
// so one pass over the row with a running m, s and w = sum e t gives everything; when
// m grows by d, s and w become s f and (w - s d it) f with f = exp(-d it).  Inside
// the kernels t is in units of ln 2 (c = it log2 e), so e = 2^t is one instruction.
//
// Gradient of  sum_j g_j log p_{id_j} + h H + z lse  with respect to x_v:
//   it [ sum_j g_j (v == id_j) + p_v (z - sum_j g_j - h H - h log p_v) ]
//
// Empty rows and odd values.  A masked logit is -inf: p = 0, and it adds nothing to w
// (t is clamped at -200, where 2^t is already 0, so no 0 * inf arises; the clamp keeps
// NaN).  A row with nothing but -inf has s = 0: lse and every log p are -inf, the
// entropy and the gradient 0.  NaN or +inf anywhere makes the row's numbers NaN; its
// top alternatives keep the sampler's order (NaN last).
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include "zs_device.cuh"

namespace zs {

constexpr int kLpMaxTop = 128;   // ZS_LOGPROBS_MAX_TOP
constexpr int kLpMaxIds = 256;   // ZS_LOGPROBS_MAX_IDS
constexpr int kLpMaxCl = 16;     // CTAs per row at most (one cluster)
constexpr int kLpCandCap = 1536; // candidates ranked at once
constexpr float kLpFloor = -200.0f;
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr double kLpLn2 = 0.6931471805599453;

struct LpRow {  // zs_logprob_row
    float max, sum, entropy, inv_temp;
};

// ---- 16-byte vectors of f32, f16 or bf16 ----
template <typename T>
struct LpVec {
    static constexpr int N = 16 / (int)sizeof(T);
};
__device__ __forceinline__ float lp_float(float v) { return v; }
__device__ __forceinline__ float lp_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void lp_unpack(const uint4& q, float (&v)[4], float) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& q, float (&v)[8], __half) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void lp_unpack(const uint4& q, float (&v)[8], __nv_bfloat16) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint4 lp_pack(const float (&v)[4], float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 lp_pack(const float (&v)[8], __half) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 lp_pack(const float (&v)[8], __nv_bfloat16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void lp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void lp_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
// A vector of -inf: what a lane without a vector reads (it changes nothing).
__device__ __forceinline__ uint4 lp_fill(float) {
    return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
__device__ __forceinline__ uint4 lp_fill(__half) {
    return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
}
__device__ __forceinline__ uint4 lp_fill(__nv_bfloat16) {
    return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}

// max(a, b) that is NaN when either is.
__device__ __forceinline__ float lp_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// n elements at p cut into an unaligned head (< N elements), nvec 16-byte vectors and a
// tail (< N elements).
struct LpCut {
    int head, nvec, tail;
};
template <typename T>
__device__ __forceinline__ LpCut lp_cut(const T* p, int n) {
    constexpr int N = LpVec<T>::N;
    const int mis = (int)(((uintptr_t)p & 15u) / sizeof(T));
    LpCut c;
    c.head = min(n, (N - mis) & (N - 1));
    c.nvec = (n - c.head) / N;
    c.tail = n - c.head - c.nvec * N;
    return c;
}

// ---- running statistics ----
struct LpStat {
    float m, s, w;  // max, sum of 2^t, sum of 2^t t with t = (x - m) c
};
__device__ __forceinline__ LpStat lp_empty() { return {-INFINITY, 0.0f, 0.0f}; }

// Moves a statistic to a larger maximum.
__device__ __forceinline__ void lp_raise(LpStat& a, float m, float c) {
    const float t = fmaxf((a.m - m) * c, kLpFloor);
    const float f = fast_exp2(t);
    a.w = f * fmaf(a.s, t, a.w);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ LpStat lp_merge(LpStat a, LpStat b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (m > a.m) lp_raise(a, m, c);
    if (m > b.m) lp_raise(b, m, c);
    a.s += b.s;
    a.w += b.w;
    return a;
}
__device__ __forceinline__ LpStat lp_warp_merge(LpStat a, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpStat b;
        b.m = __shfl_xor_sync(kFull, a.m, o);
        b.s = __shfl_xor_sync(kFull, a.s, o);
        b.w = __shfl_xor_sync(kFull, a.w, o);
        a = lp_merge(a, b, c);
    }
    return a;
}
__device__ __forceinline__ void lp_add(LpStat& a, float v, float base, float c) {
    const float t = lp_max_nan((v - base) * c, kLpFloor);
    const float e = fast_exp2(t);
    a.s += e;
    a.w = fmaf(e, t, a.w);
}
__device__ __forceinline__ void lp_scalar(LpStat& a, float v, float c) {
    if (v > a.m) lp_raise(a, v, c);
    lp_add(a, v, a.m == -INFINITY ? 0.0f : a.m, c);
}

// 1 / temp as the sampler takes it (1 for greedy rows).
__device__ __forceinline__ float lp_inv_temp(float temp, const float* row_temp, int64_t row) {
    const float t = row_temp ? row_temp[row] : temp;
    return t <= 0.0f ? 1.0f : 1.0f / t;
}

// log p of a value from the row's statistics, in f64 (one value per row and id).
__device__ __forceinline__ float lp_value(float x, float m, double log_s, float it) {
    if (log_s == -INFINITY) return -INFINITY;
    return (float)(((double)x - (double)m) * (double)it - log_s);
}
__device__ __forceinline__ float lp_entropy(const LpStat& a, double log_s) {
    if (a.s == 0.0f) return 0.0f;
    const float h = (float)(log_s - kLpLn2 * (double)a.w / (double)a.s);
    return h < 0.0f ? 0.0f : h;
}

struct LpArgs {
    const void* logits;
    int64_t ld;
    int32_t B, n;
    float temp;
    const float* row_temp;
    const int32_t* ids;  // [B][ids_ld]
    int64_t ids_ld;
    int32_t n_ids;
    int32_t k;           // alternatives per row, at most n
    int32_t top_ld;
    float* out_logp;     // [B][n_ids]
    int32_t* top_ids;    // [B][top_ld]
    float* top_logp;
    float* out_entropy;  // [B], optional
    float* out_lse;      // [B], optional
    LpRow* out_rows;     // [B], optional
    int32_t cl;          // CTAs per row
};

// Number of keys of a descending list that are greater than `key`.
__device__ __forceinline__ int lp_above(const uint64_t* list, int n, uint64_t key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > key)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

// The 32 keys of a warp in descending order (bitonic).
__device__ __forceinline__ void lp_warp_sort(uint64_t& key, uint32_t& tag, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const uint64_t ok = __shfl_xor_sync(kFull, key, o);
            const uint32_t ot = __shfl_xor_sync(kFull, tag, o);
            const bool lower = (lane & o) == 0;
            const bool desc = (lane & size) == 0 || size == 32;
            const bool take = (lower == desc) ? ok > key : ok < key;
            if (take) {
                key = ok;
                tag = ot;
            }
        }
    }
}

template <int NT>
struct LpTopSmem {
    uint64_t warp_keys[NT];               // each warp's sorted thread keys
    uint32_t warp_tags[NT];
    uint64_t cta_keys[kLpMaxTop];         // this CTA's best, read by the leader
    uint32_t cta_tags[kLpMaxTop];
    uint64_t all_keys[kLpMaxCl * kLpMaxTop];
    uint32_t all_tags[kLpMaxCl * kLpMaxTop];
    uint64_t sel_keys[kLpMaxTop];
    uint32_t sel_tags[kLpMaxTop];         // source CTA << 16 | thread
    uint64_t cand[kLpCandCap];
    uint64_t red[NT / 32];
    int ncta, nsel, ncand;
};

// One row per cluster of a.cl CTAs (one CTA when a.cl is 1).  The row is streamed
// once with 16-byte loads, kUnroll in flight per thread; the CTAs' statistics meet in
// the leader (rank 0) through distributed shared memory in rank order, so no scratch,
// no atomics and a fixed summation order.
//
// Alternatives (TOP).  Each thread's elements form a group whose best key (value
// desc, id asc) the running maximum already gives, up to the vector it was first seen
// in.  The k best elements all lie in the k groups with the best such keys: if an
// element's group is not among them, k groups rank before it and each holds an element
// that does.  So the pass keeps one position per thread, the k best groups are found
// at the end (warp sort, then ranks by binary search), and only those k groups (a
// few hundred elements) are read again, from L2.  Should the candidates not suffice
// (NaN groups) or not fit, the leader takes the k best one after another from the row.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT) zs_logprobs_kernel(const LpArgs a) {
    namespace cg = cooperative_groups;
    constexpr int N = LpVec<T>::N;
    constexpr int kUnroll = 4;
    extern __shared__ __align__(16) uint8_t lp_raw[];
    __shared__ LpStat warp_stat[NT / 32];
    __shared__ LpStat cta_stat;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = a.cl > 1 ? (int)cluster.block_rank() : 0;
    const int64_t row = blockIdx.x / a.cl;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
    const float it = lp_inv_temp(a.temp, a.row_temp, row);
    const float c = it * kLpLog2e;

    const LpCut cut = lp_cut(x, a.n);
    const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
    const int v0 = (int)((int64_t)cut.nvec * rank / a.cl);
    const int v1 = (int)((int64_t)cut.nvec * (rank + 1) / a.cl);

    LpStat st = lp_empty();
    int pos = -1;  // first id of the vector that holds this thread's maximum
    if (rank == 0 && tid < cut.head) {
        lp_scalar(st, lp_float(x[tid]), c);
        pos = tid;
    }
    if (TOP && pos < 0 && v0 + tid < v1) pos = cut.head + (v0 + tid) * N;
    for (int i = v0 + tid; i < v1; i += NT * kUnroll) {
        uint4 q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            q[u] = i + u * NT < v1 ? __ldcs(xv + i + u * NT) : lp_fill(T());
        float m = st.m;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float v[N];
            lp_unpack(q[u], v, T());
            float b = v[0];
#pragma unroll
            for (int j = 1; j < N; ++j) b = fmaxf(b, v[j]);
            if (b > m) {
                m = b;
                if (TOP) pos = cut.head + (i + u * NT) * N;
            }
        }
        if (m > st.m) lp_raise(st, m, c);
        const float base = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float v[N];
            lp_unpack(q[u], v, T());
#pragma unroll
            for (int j = 0; j < N; ++j) lp_add(st, v[j], base, c);
        }
    }
    if (rank == a.cl - 1 && tid < cut.tail) {
        const int id = cut.head + cut.nvec * N + tid;
        const float v = lp_float(x[id]);
        if (TOP && (pos < 0 || v > st.m)) pos = id;
        lp_scalar(st, v, c);
    }
    const float best = st.m;  // this thread's own maximum

    // ---- statistics: warp, CTA, cluster ----
    st = lp_warp_merge(st, c);
    if (lane == 0) warp_stat[warp] = st;
    __syncthreads();
    if (warp == 0) {
        LpStat t = lane < NT / 32 ? warp_stat[lane] : lp_empty();
        t = lp_warp_merge(t, c);
        if (lane == 0) cta_stat = t;
    }

    LpTopSmem<NT>& tp = *reinterpret_cast<LpTopSmem<NT>*>(lp_raw);
    const int k = a.k;
    if (TOP) {
        // this CTA's k best groups
        uint64_t key = pos >= 0 ? make_key(best, pos) : 0ull;
        uint32_t tag = (uint32_t)tid;
        lp_warp_sort(key, tag, lane);
        tp.warp_keys[tid] = key;
        tp.warp_tags[tid] = tag;
        if (tid == 0) {
            tp.ncta = 0;
            tp.ncand = 0;
        }
        __syncthreads();
        if (key != 0ull) {
            int r = lane;
            for (int w = 0; w < NT / 32 && r < k; ++w)
                if (w != warp) r += lp_above(tp.warp_keys + w * 32, 32, key);
            if (r < k) {
                tp.cta_keys[r] = key;
                tp.cta_tags[r] = tag;
                atomicAdd(&tp.ncta, 1);
            }
        }
    }
    if (a.cl > 1)
        cluster.sync();
    else
        __syncthreads();
    if (rank != 0) {
        cluster.sync();  // the leader has read this CTA's shared memory
        return;
    }

    st = cta_stat;
    if (a.cl > 1) {
        st = lane < a.cl ? *cluster.map_shared_rank(&cta_stat, lane) : lp_empty();
        st = lp_warp_merge(st, c);
    }
    if (TOP) {
        // the row's k best groups
        const int cl = a.cl;
        int total = 0;
        for (int r = 0; r < cl; ++r) {
            const LpTopSmem<NT>* o = cl > 1 ? cluster.map_shared_rank(&tp, r) : &tp;
            const int nr = o->ncta;
            total += nr;
            for (int i = tid; i < k; i += NT) {
                tp.all_keys[r * k + i] = i < nr ? o->cta_keys[i] : 0ull;
                tp.all_tags[r * k + i] = i < nr ? ((uint32_t)r << 16) | o->cta_tags[i] : 0u;
            }
        }
        const int nsel = min(k, total);
        if (cl > 1)
            cluster.sync();
        else
            __syncthreads();
        for (int i = tid; i < cl * k; i += NT) {
            const uint64_t key = tp.all_keys[i];
            if (key == 0ull) continue;
            int r = i % k;
            for (int o = 0; o < cl && r < nsel; ++o)
                if (o != i / k) r += lp_above(tp.all_keys + o * k, k, key);
            if (r < nsel) {
                tp.sel_keys[r] = key;
                tp.sel_tags[r] = tp.all_tags[i];
            }
        }
        __syncthreads();
        // Every element at or above the last group's best is a candidate; its key is
        // known up to the id within its vector.
        uint64_t floor_key = 0ull;
        if (nsel == k) {
            const uint64_t last = tp.sel_keys[k - 1];
            const int id = key_id(last);
            const int span = (id >= cut.head && id < cut.head + cut.nvec * N) ? N : 1;
            floor_key = (last & 0xffffffff00000000ull) | (uint64_t)(~(uint32_t)(id + span - 1));
        }
        auto offer = [&](float v, int id) {
            const uint64_t key = make_key(v, id);
            if (key >= floor_key) {
                const int at = atomicAdd(&tp.ncand, 1);
                if (at < kLpCandCap) tp.cand[at] = key;
            }
        };
        for (int g = warp; g < nsel; g += NT / 32) {
            const int src = (int)(tp.sel_tags[g] >> 16), t = (int)(tp.sel_tags[g] & 0xffffu);
            const int b0 = (int)((int64_t)cut.nvec * src / cl);
            const int b1 = (int)((int64_t)cut.nvec * (src + 1) / cl);
            for (int i = b0 + t + lane * NT; i < b1; i += 32 * NT) {
                const uint4 q = xv[i];
                float v[N];
                lp_unpack(q, v, T());
#pragma unroll
                for (int j = 0; j < N; ++j) offer(v[j], cut.head + i * N + j);
            }
            if (lane == 0 && src == 0 && t < cut.head) offer(lp_float(x[t]), t);
            if (lane == 0 && src == cl - 1 && t < cut.tail) {
                const int id = cut.head + cut.nvec * N + t;
                offer(lp_float(x[id]), id);
            }
        }
        __syncthreads();
        const int nc = tp.ncand;
        const double log_s = log((double)st.s) + 0.0;
        const double ls = st.s == 0.0f ? -INFINITY : log_s;
        auto put = [&](int r, uint64_t key) {
            const int id = key_id(key);
            a.top_ids[row * a.top_ld + r] = id;
            a.top_logp[row * a.top_ld + r] = lp_value(lp_float(x[id]), st.m, ls, it);
        };
        if (nc >= k && nc <= kLpCandCap) {
            for (int i = tid; i < nc; i += NT) {
                const uint64_t key = tp.cand[i];
                int r = 0;
                for (int j = 0; j < nc && r < k; ++j) r += tp.cand[j] > key ? 1 : 0;
                if (r < k) put(r, key);
            }
        } else {
            uint64_t prev = ~0ull;
            for (int r = 0; r < k; ++r) {
                uint64_t b = 0ull;
                for (int i = tid; i < a.n; i += NT) {
                    const uint64_t key = make_key(lp_float(x[i]), i);
                    if (key < prev && key > b) b = key;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t t = __shfl_xor_sync(kFull, b, o);
                    b = t > b ? t : b;
                }
                if (lane == 0) tp.red[warp] = b;
                __syncthreads();
                b = tp.red[0];
                for (int w = 1; w < NT / 32; ++w) b = tp.red[w] > b ? tp.red[w] : b;
                __syncthreads();
                if (tid == 0) put(r, b);
                prev = b;
            }
        }
    } else if (a.cl > 1) {
        cluster.sync();
    }

    // ---- the row's numbers ----
    const double log_s = st.s == 0.0f ? -INFINITY : log((double)st.s);
    for (int j = tid; j < a.n_ids; j += NT) {
        const int32_t id = a.ids[row * a.ids_ld + j];
        a.out_logp[row * a.n_ids + j] =
            (id < 0 || id >= a.n) ? 0.0f : lp_value(lp_float(x[id]), st.m, log_s, it);
    }
    if (tid == 0) {
        const float h = lp_entropy(st, log_s);
        if (a.out_entropy) a.out_entropy[row] = h;
        if (a.out_lse)
            a.out_lse[row] = st.s == 0.0f ? -INFINITY : (float)((double)st.m * (double)it + log_s);
        if (a.out_rows) a.out_rows[row] = {st.m, st.s, h, it};
    }
}

// ---- gradient ----
struct LpBackArgs {
    const void* logits;
    int64_t ld;
    int32_t B, n;
    const LpRow* rows;
    const int32_t* ids;
    int64_t ids_ld;
    int32_t n_ids;
    const float* g_logp;     // [B][n_ids], optional
    const float* g_entropy;  // [B], optional
    const float* g_lse;      // [B], optional
    void* grad;
    int64_t grad_ld;
    int32_t chunks;          // CTAs per row
};

constexpr int kLpBackThreads = 256;
constexpr int kLpBackUnroll = 4;
template <typename T>
__host__ __device__ constexpr int lp_back_chunk() {  // elements per CTA
    return kLpBackThreads * LpVec<T>::N * kLpBackUnroll * 2;
}

// One CTA per chunk of a row: p is recomputed from the row's maximum and sum, so
// the pass reads the logits once and writes the gradient once.  The given ids of the
// chunk are written again behind the chunk, each by one thread that adds the
// gradients of all its occurrences in order.  The gradient may be the logits' buffer.
template <typename T>
__global__ void __launch_bounds__(kLpBackThreads, 4) zs_logprobs_backward_kernel(const LpBackArgs a) {
    constexpr int N = LpVec<T>::N;
    constexpr int NT = kLpBackThreads;
    const int64_t row = blockIdx.x / a.chunks;
    const int ch = (int)(blockIdx.x - row * a.chunks);
    const int tid = threadIdx.x, lane = tid & 31;
    const int e0 = ch * lp_back_chunk<T>();
    const int cnt = min(a.n - e0, lp_back_chunk<T>());
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld + e0;
    T* gx = reinterpret_cast<T*>(a.grad) + row * a.grad_ld + e0;
    const LpRow rw = a.rows[row];
    const bool dead = rw.sum == 0.0f;
    const float c = rw.inv_temp * kLpLog2e;

    // sum of the given tokens' gradients (every warp the same order)
    float g = 0.0f;
    if (a.g_logp) {
        for (int j = lane; j < a.n_ids; j += 32) {
            const int32_t id = a.ids[row * a.ids_ld + j];
            if (id >= 0 && id < a.n) g += a.g_logp[row * a.n_ids + j];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) g += __shfl_xor_sync(kFull, g, o);
    }
    const float gh = a.g_entropy ? a.g_entropy[row] : 0.0f;
    const float gz = a.g_lse ? a.g_lse[row] : 0.0f;
    const double log_s = dead ? 0.0 : log((double)rw.sum);
    // p (z - g - h H - h log p) it = e (ca + cb t), log p = ln 2 t - ln s
    const float inv_s = dead ? 0.0f : 1.0f / rw.sum;
    const float ca = (float)((double)rw.inv_temp *
                             ((double)gz - (double)g - (double)gh * ((double)rw.entropy - log_s))) * inv_s;
    const float cb = (float)(-(double)rw.inv_temp * (double)gh * kLpLn2) * inv_s;
    const float base = rw.max;
    auto grad_of = [&](float v) {
        const float t = lp_max_nan((v - base) * c, kLpFloor);
        return dead ? 0.0f : fast_exp2(t) * fmaf(cb, t, ca);
    };

    // this thread's given id, read before the chunk is overwritten
    float fix = 0.0f;
    int fix_at = -1;
    if (a.g_logp && tid < a.n_ids) {
        const int32_t id = a.ids[row * a.ids_ld + tid];
        if (id >= e0 && id < e0 + cnt && !dead) {
            bool first = true;
            for (int j = 0; j < tid; ++j) first = first && a.ids[row * a.ids_ld + j] != id;
            if (first) {
                float gs = 0.0f;
                for (int j = tid; j < a.n_ids; ++j)
                    if (a.ids[row * a.ids_ld + j] == id) gs += a.g_logp[row * a.n_ids + j];
                fix = fmaf(rw.inv_temp, gs, grad_of(lp_float(x[id - e0])));
                fix_at = id - e0;
            }
        }
    }
    __syncthreads();

    if ((((uintptr_t)x ^ (uintptr_t)gx) & 15u) == 0) {
        const LpCut cut = lp_cut(x, cnt);
        const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
        uint4* gv = reinterpret_cast<uint4*>(gx + cut.head);
        for (int i = tid; i < cut.nvec; i += NT * kLpBackUnroll) {
            uint4 q[kLpBackUnroll];
#pragma unroll
            for (int u = 0; u < kLpBackUnroll; ++u)
                if (i + u * NT < cut.nvec) q[u] = __ldcs(xv + i + u * NT);
#pragma unroll
            for (int u = 0; u < kLpBackUnroll; ++u) {
                if (i + u * NT < cut.nvec) {
                    float v[N];
                    lp_unpack(q[u], v, T());
#pragma unroll
                    for (int j = 0; j < N; ++j) v[j] = grad_of(v[j]);
                    __stcs(gv + i + u * NT, lp_pack(v, T()));
                }
            }
        }
        if (tid < cut.head) lp_store(gx + tid, grad_of(lp_float(x[tid])));
        const int t0 = cut.head + cut.nvec * N;
        if (tid < cut.tail) lp_store(gx + t0 + tid, grad_of(lp_float(x[t0 + tid])));
    } else {
        // rows of the two buffers start at different offsets from a 16-byte boundary
        for (int i = tid; i < cnt; i += NT) lp_store(gx + i, grad_of(lp_float(x[i])));
    }
    __syncthreads();
    if (fix_at >= 0) lp_store(gx + fix_at, fix);
}

}  // namespace zs
