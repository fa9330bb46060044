// zs_embed.cuh -- rows of the embedding table (scaled), and the table's gradient
// summed per token id.
//
//   out[i]        = scale * table[ids[i]]              (0 for an id outside the table)
//   grad_table[v] = scale * sum_{i: ids[i] == v} grad_out[i]
//
// The gradient is taken by sorted tokens: (id, position) pairs are sorted (stable), and
// each id's rows are summed in f32 in the order of their positions, chunk by chunk, so
// the result does not depend on timing and each table row is rounded once.
#pragma once

#include <cooperative_groups.h>
#include <stdint.h>

#include "zs_device.cuh"
#include "zs_logprobs.cuh"

namespace zs {

// A granule: G consecutive elements, 16 bytes of the narrower of the two types.
template <typename A, typename B>
struct EmGran {
    static constexpr int G = (sizeof(A) == 2 || sizeof(B) == 2) ? 8 : 4;
};

template <int G>
__device__ __forceinline__ void em_load(const float* p, float (&v)[G]) {
#pragma unroll
    for (int i = 0; i < G; i += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + i));
        v[i] = q.x;
        v[i + 1] = q.y;
        v[i + 2] = q.z;
        v[i + 3] = q.w;
    }
}
template <int G, typename T>
__device__ __forceinline__ void em_load(const T* p, float (&v)[G]) {
    static_assert(G == 8 && sizeof(T) == 2, "one 16-byte load");
    lp_unpack(__ldg(reinterpret_cast<const uint4*>(p)), v, T());
}
// Loads from memory this kernel also writes (not the read-only path).
template <int G, typename T>
__device__ __forceinline__ void em_load_rw(const T* p, float (&v)[G]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < G; i += 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + i);
            v[i] = q.x;
            v[i + 1] = q.y;
            v[i + 2] = q.z;
            v[i + 3] = q.w;
        }
    } else {
        lp_unpack(*reinterpret_cast<const uint4*>(p), v, T());
    }
}
template <int G>
__device__ __forceinline__ void em_store(float* p, const float (&v)[G]) {
#pragma unroll
    for (int i = 0; i < G; i += 4)
        *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int G, typename T>
__device__ __forceinline__ void em_store(T* p, const float (&v)[G]) {
    *reinterpret_cast<uint4*>(p) = lp_pack(v, T());
}

// ---- lookup ----
struct EmArgs {
    const void* table;
    int64_t table_ld;
    int32_t V, E;
    const int32_t* ids;
    int64_t n;
    float scale;
    void* out;
    int64_t out_ld;
    int32_t tpr;  // threads per row: a power of two, 32 to kEmThreads
};
constexpr int kEmThreads = 256;

// kEmThreads / tpr rows at a time, U of them per thread, so that U id loads and then
// U row loads are in flight.  VEC: every row of both buffers starts at a 16-byte
// boundary; else one element per thread and step.
template <typename TI, typename TO, int U, bool VEC>
__global__ void __launch_bounds__(kEmThreads) zs_embed_kernel(const EmArgs a) {
    constexpr int G = VEC ? EmGran<TI, TO>::G : 1;
    const int rows_at_once = kEmThreads / a.tpr;
    const int sub = threadIdx.x / a.tpr, lane = threadIdx.x & (a.tpr - 1);
    const int64_t i0 = (int64_t)blockIdx.x * rows_at_once * U + sub;
    const TI* table = reinterpret_cast<const TI*>(a.table);
    TO* out = reinterpret_cast<TO*>(a.out);
    int32_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + (int64_t)u * rows_at_once;
        id[u] = i < a.n ? __ldg(a.ids + i) : -1;
        if (id[u] >= a.V) id[u] = -1;
    }
    const int full = a.E / G;
    for (int g = lane; g < full; g += a.tpr) {
        float v[U][G];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < G; ++j) v[u][j] = 0.0f;
            if (id[u] >= 0) {
                const TI* p = table + (int64_t)id[u] * a.table_ld + (int64_t)g * G;
                if constexpr (VEC)
                    em_load(p, v[u]);
                else
                    v[u][0] = lp_float(*p);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + (int64_t)u * rows_at_once;
            if (i >= a.n) continue;
            TO* p = out + i * a.out_ld + (int64_t)g * G;
#pragma unroll
            for (int j = 0; j < G; ++j) v[u][j] = id[u] >= 0 ? v[u][j] * a.scale : 0.0f;
            if constexpr (VEC)
                em_store(p, v[u]);
            else
                lp_store(p, v[u][0]);
        }
    }
    if constexpr (VEC) {  // the last E mod G columns
        const int e = full * G + lane;
        if (lane < G && e < a.E) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = i0 + (int64_t)u * rows_at_once;
                if (i >= a.n) continue;
                lp_store(out + i * a.out_ld + e,
                         id[u] >= 0 ? lp_float(table[(int64_t)id[u] * a.table_ld + e]) * a.scale : 0.0f);
            }
        }
    }
}

// ---- gradient: sort ----
constexpr int kEsCl = 8;          // CTAs that sort (one portable cluster)
constexpr int kEsThreads = 1024;
constexpr int kEsWarps = kEsThreads / 32;
constexpr int kEsMaxBins = 512;
constexpr int kEsChunk = 32;      // sorted positions per CTA of the summing kernel

struct EsSmem {
    uint32_t hist[kEsWarps][kEsMaxBins];
    uint32_t tot[kEsMaxBins];   // this CTA's digit counts, read by the others
    uint32_t base[kEsMaxBins];
    uint32_t scan[kEsWarps];
};

struct EsArgs {
    const int32_t* ids;
    int32_t n, V;
    int32_t digit_bits, passes;
    uint32_t* key[2];  // ping-pong; the last pass writes [passes & 1]
    uint32_t* pos[2];
    // zero fill by the other clusters: zrows rows of zcols elements of zsize bytes,
    // zld elements apart (zrows 0: none)
    uint8_t* z;
    int64_t zrows, zcols, zld;
    int32_t zsize;
};

// Zeroes bytes [0, bytes) at p (an element boundary) with the threads of `tid` of `nt`.
__device__ __forceinline__ void es_zero(uint8_t* p, int64_t bytes, int64_t tid, int64_t nt) {
    const int64_t head = min(bytes, (int64_t)((16u - ((uintptr_t)p & 15u)) & 15u));
    const int64_t nvec = (bytes - head) >> 4;
    const int64_t tail = bytes - head - (nvec << 4);
    uint4* v = reinterpret_cast<uint4*>(p + head);
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    int64_t i = tid;
    for (; i + 3 * nt < nvec; i += 4 * nt) {
        __stcs(v + i, z);
        __stcs(v + i + nt, z);
        __stcs(v + i + 2 * nt, z);
        __stcs(v + i + 3 * nt, z);
    }
    for (; i < nvec; i += nt) __stcs(v + i, z);
    if (tid < head) p[tid] = 0;
    if (tid < tail) p[head + (nvec << 4) + tid] = 0;
}

// Cluster 0 sorts the n (id, position) pairs by id, stable, least significant digit
// first; an id outside the table becomes V and sorts last.  The other clusters zero
// the table meanwhile.  Per pass each warp counts the digits of its contiguous share;
// a digit's place is the count of smaller digits, of earlier CTAs', of earlier warps'
// and of earlier items of the warp (by __match_any_sync), all of them exact counts, so
// the order is fixed.  The pairs stay in L2 between passes.
__global__ void __launch_bounds__(kEsThreads, 1) zs_embed_sort_kernel(const EsArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t es_raw[];
    EsSmem& sm = *reinterpret_cast<EsSmem*>(es_raw);
    grid_dep_trigger();  // the summing kernel may be scheduled; it waits for this grid
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (blockIdx.x >= kEsCl) {
        const int64_t z = blockIdx.x - kEsCl, nz = gridDim.x - kEsCl;
        if (a.zrows == 1) {
            es_zero(a.z, a.zcols * a.zsize, z * kEsThreads + tid, nz * kEsThreads);
        } else {
            for (int64_t r = z; r < a.zrows; r += nz)
                es_zero(a.z + r * a.zld * a.zsize, a.zcols * a.zsize, tid, kEsThreads);
        }
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank();
    constexpr int kStep = kEsCl * kEsWarps * 32;
    const int per = (int)(((int64_t)a.n + kStep - 1) / kStep) * 32;  // items per warp
    const int64_t w0 = (int64_t)(rank * kEsWarps + warp) * per;
    const int lo = (int)min((int64_t)a.n, w0), hi = (int)min((int64_t)a.n, w0 + per);
    const int bins = 1 << a.digit_bits;
    const uint32_t mask = (uint32_t)bins - 1u;
    for (int p = 0; p < a.passes; ++p) {
        const int shift = p * a.digit_bits;
        const uint32_t* src_k = a.key[p & 1];
        const uint32_t* src_p = a.pos[p & 1];
        uint32_t* dst_k = a.key[(p + 1) & 1];
        uint32_t* dst_p = a.pos[(p + 1) & 1];
        auto key_at = [&](int i) -> uint32_t {
            if (p > 0) return __ldcg(src_k + i);
            const int32_t id = a.ids[i];
            return id < 0 || id >= a.V ? (uint32_t)a.V : (uint32_t)id;
        };
        for (int i = tid; i < kEsWarps * kEsMaxBins; i += kEsThreads) (&sm.hist[0][0])[i] = 0u;
        __syncthreads();
        for (int i = lo + lane; i < hi; i += 32)
            atomicAdd(&sm.hist[warp][(key_at(i) >> shift) & mask], 1u);
        __syncthreads();
        // per digit: counts of earlier warps, and the CTA's total
        uint32_t mine = 0;
        if (tid < bins) {
#pragma unroll 8
            for (int w = 0; w < kEsWarps; ++w) {
                const uint32_t h = sm.hist[w][tid];
                sm.hist[w][tid] = mine;
                mine += h;
            }
            sm.tot[tid] = mine;
        }
        cluster.sync();
        uint32_t all = 0, before = 0;
        if (tid < bins) {
#pragma unroll
            for (int r = 0; r < kEsCl; ++r) {
                const uint32_t t = cluster.map_shared_rank(&sm, r)->tot[tid];
                before += r < rank ? t : 0u;
                all += t;
            }
        }
        // exclusive prefix of `all` over the digits
        uint32_t inc = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(kFull, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) sm.scan[warp] = inc;
        __syncthreads();
        uint32_t off = 0;
        for (int w = 0; w < warp; ++w) off += sm.scan[w];
        if (tid < bins) sm.base[tid] = off + inc - all + before;
        __syncthreads();
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            const bool live = i < hi;
            const uint32_t k = live ? key_at(i) : 0u;
            const uint32_t d = live ? (k >> shift) & mask : 0xffffffffu;
            const unsigned same = __match_any_sync(kFull, d);
            const int r = __popc(same & lanemask_lt());
            uint32_t at = 0;
            if (live) at = sm.hist[warp][d] + (uint32_t)r + sm.base[d];
            __syncwarp();
            if (live && r == 0) sm.hist[warp][d] += (uint32_t)__popc(same);
            __syncwarp();
            if (live) {
                dst_k[at] = k;
                dst_p[at] = p > 0 ? __ldcg(src_p + i) : (uint32_t)i;
            }
        }
        // every CTA's pairs of this pass are written, and every CTA has read the totals
        __threadfence();
        cluster.sync();
    }
}

// ---- gradient: sum ----
struct EbArgs {
    const void* grad;
    int64_t grad_ld;
    int32_t n, V, E;
    const uint32_t* key;  // sorted ids
    const uint32_t* pos;
    float scale;
    void* table;
    int64_t table_ld;
    int32_t accumulate;
    float* part;          // [chunks][2][E]: the run that came in, the run that goes on
    int32_t chunks;
};

template <typename TG, typename TT, bool VEC, int G>
__device__ __forceinline__ void eb_write(const EbArgs& a, uint32_t id, int col, float (&acc)[G]) {
    TT* p = reinterpret_cast<TT*>(a.table) + (int64_t)id * a.table_ld + col;
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < G; ++j) acc[j] *= a.scale;
        if (a.accumulate) {
            float old[G];
            em_load_rw(p, old);
#pragma unroll
            for (int j = 0; j < G; ++j) acc[j] += old[j];
        }
        em_store(p, acc);
    } else {
        float v = acc[0] * a.scale;
        if (a.accumulate) v += lp_float(*p);
        lp_store(p, v);
    }
}

// One CTA sums kEsChunk sorted positions, a granule of columns per thread.  A run of
// equal ids inside the chunk is finished here; one that crosses its borders leaves a
// partial sum for zs_embed_join_kernel.
template <typename TG, typename TT, bool VEC>
__global__ void __launch_bounds__(128) zs_embed_sum_kernel(const EbArgs a) {
    constexpr int G = VEC ? EmGran<TG, TT>::G : 1;
    constexpr int kAhead = 8;  // rows in flight
    __shared__ uint32_t keys[kEsChunk + 2];  // [0] before the chunk, then the chunk, then after
    __shared__ uint32_t poss[kEsChunk];
    grid_dep_trigger();
    grid_dep_wait();  // the sorted pairs
    const int s0 = blockIdx.x * kEsChunk;
    const int cnt = min(kEsChunk, a.n - s0);
    const uint32_t none = 0xffffffffu;  // not an id: those are below 2^31
    for (int i = threadIdx.x; i < kEsChunk + 2; i += blockDim.x) {
        const int p = s0 + i - 1;
        keys[i] = (p >= 0 && p < a.n) ? a.key[p] : none;
        if (i < cnt) poss[i] = a.pos[s0 + i];
    }
    __syncthreads();
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * G;
    if (col >= a.E) return;
    const TG* grad = reinterpret_cast<const TG*>(a.grad) + col;
    float acc[G];
#pragma unroll
    for (int j = 0; j < G; ++j) acc[j] = 0.0f;
    bool came_in = keys[0] == keys[1];  // the current run began in an earlier chunk
    for (int i0 = 0; i0 < cnt; i0 += kAhead) {
        float v[kAhead][G];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u < cnt && keys[i0 + u + 1] < (uint32_t)a.V) {
                const TG* p = grad + (int64_t)poss[i0 + u] * a.grad_ld;
                if constexpr (VEC)
                    em_load(p, v[u]);
                else
                    v[u][0] = lp_float(*p);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            if (i >= cnt) break;
            const uint32_t id = keys[i + 1];
            if (id >= (uint32_t)a.V) break;  // ids outside the table sort last
#pragma unroll
            for (int j = 0; j < G; ++j) acc[j] += v[u][j];
            const bool ends = keys[i + 2] != id;
            if (ends || i + 1 == cnt) {
                if (ends && !came_in) {
                    eb_write<TG, TT, VEC>(a, id, col, acc);
                } else {
                    float* p = a.part + ((int64_t)blockIdx.x * 2 + (came_in ? 0 : 1)) * a.E + col;
#pragma unroll
                    for (int j = 0; j < G; ++j) p[j] = acc[j];
                }
#pragma unroll
                for (int j = 0; j < G; ++j) acc[j] = 0.0f;
                came_in = false;
            }
        }
    }
}

// Finishes the runs that cross chunk borders: the CTA that has the chunk in which such
// a run begins adds the run's partial sums, group y of its kEjGroups every kEjGroups-th
// of them in order, then the groups in order.
constexpr int kEjGroups = 8;
template <typename TG, typename TT, bool VEC>
__global__ void __launch_bounds__(128 * kEjGroups) zs_embed_join_kernel(const EbArgs a) {
    constexpr int G = VEC ? EmGran<TG, TT>::G : 1;
    extern __shared__ float ej_part[];  // [kEjGroups][blockDim.x][G]
    __shared__ int list[128 * kEjGroups];
    __shared__ int nlist;
    grid_dep_wait();
    const int nt = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * G;
    for (int c0 = blockIdx.x; c0 < a.chunks; c0 += gridDim.x * nt) {
        // which of this CTA's next nt chunks start a crossing run
        if (tid == 0) nlist = 0;
        __syncthreads();
        const int64_t c = c0 + (int64_t)tid * gridDim.x;
        if (c < a.chunks - 1) {
            const int64_t s0 = c * kEsChunk, s1 = s0 + kEsChunk;  // s1 < n
            const uint32_t k = a.key[s1];
            const bool crosses = k < (uint32_t)a.V && a.key[s1 - 1] == k;
            if (crosses && (a.key[s0] != k || s0 == 0 || a.key[s0 - 1] != k))
                list[atomicAdd(&nlist, 1)] = (int)c;
        }
        __syncthreads();
        const int nl = nlist;
        for (int l = 0; l < nl; ++l) {
            const int ch = list[l];
            const uint32_t k = a.key[(int64_t)(ch + 1) * kEsChunk];
            // chunks after ch whose first position belongs to the run
            int m = 0;
            for (;;) {
                const int64_t at = (int64_t)(ch + 1 + m + tid) * kEsChunk;
                const int got = __syncthreads_count(at < a.n && a.key[at] == k);
                m += got;
                if (got < nt) break;
            }
            float acc[G];
#pragma unroll
            for (int j = 0; j < G; ++j) acc[j] = 0.0f;
            if (col < a.E) {
#pragma unroll 8
                for (int i = threadIdx.y; i <= m; i += kEjGroups) {
                    const float* p = a.part + ((int64_t)(ch + i) * 2 + (i == 0 ? 1 : 0)) * a.E + col;
#pragma unroll
                    for (int j = 0; j < G; ++j) acc[j] += p[j];
                }
            }
            float* mine = ej_part + ((int)threadIdx.y * blockDim.x + threadIdx.x) * G;
#pragma unroll
            for (int j = 0; j < G; ++j) mine[j] = acc[j];
            __syncthreads();
            if (threadIdx.y == 0 && col < a.E) {
                for (int y = 1; y < kEjGroups; ++y)
#pragma unroll
                    for (int j = 0; j < G; ++j)
                        acc[j] += ej_part[(y * blockDim.x + threadIdx.x) * G + j];
                eb_write<TG, TT, VEC>(a, k, col, acc);
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

}  // namespace zs
