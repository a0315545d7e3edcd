// Drawing with a row held in the shared memory of a cluster of CTAs (draw.cuh has the definition and the arithmetic).
//
// The logits are read from global memory once, with their maximum; everything else works on shared memory.  The cut that top-k and top-p make is
// found without sorting the row:
//   list    Every thread keeps the largest of its own logits.  The k-th largest of a CTA's 512 such maxima is a lower bound of the row's k-th largest
//           logit, and so is the smallest over the CTAs of the (k / CTAs)-th; the logits from the larger of the two on are collected (k and a few more),
//           sorted by value and index, and the cut lies among them.  With top-p and no top-k the 256 largest are tried first: their weight tells
//           whether the cut lies among them.
//   region  Otherwise a histogram of (max - l) in 2048 linear bins says near which bin the cut lies; the logits of that bin and its neighbours are
//           collected and sorted, the weight of all larger ones is summed exactly, and the sums tell whether the cut is there.
//   neither Where the collection would not fit 1024 entries (many equal logits) one CTA does the row by radix passes (dw_row_plain).
// Without top-k and top-p no cut is needed: min-p's is a value that follows from the maximum.
//
// The draw: sums of the kept weights per warp, whose logits follow each other in the vocabulary, then the one warp's stretch again, split over the CTA.
#pragma once
#include "draw.cuh"
#include "tc_ptx.cuh"

namespace rsv {

constexpr int kDcList = 1024;     // entries of a collection: two per thread
constexpr int kDcBins = 2048;     // four per thread
constexpr int kDcFastK = 384;     // most thread maxima asked for, of 512
constexpr int kDcTryK = 256;      // entries tried for top-p alone
constexpr int kDcMaxCtas = 8;
constexpr int kDcSliceBytes = 64 * 1024;

struct DcShared {
    // read by the other CTAs
    alignas(16) u64 list[kDcList];  // key << 32 | ~index
    union {
        uint32_t hist[kDcBins];
        u64 keys[kDcList];  // the collections of all CTAs, sorted (this CTA's own copy)
    };
    u64 seg[kDwWarps];  // kept weight of every warp's stretch
    u64 total, mass;    // weight of the slice, and of its collection
    float mx, thr_all, thr_part;
    int nan, n_list, n_above;
    // this CTA's own
    double tab[16];
    u64 wsum[kDwWarps], segs[kDcMaxCtas * kDwWarps];
    float red[kDwWarps], redmin[kDwWarps];
    uint32_t wcnt[kDwWarps], tmhist[256], first, key_all, key_part;
    int cross_all, cross_part, bin, found;
};

__device__ __forceinline__ uint32_t dc_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void dc_sync(int S) {
    if (S == 1) {
        __syncthreads();
    } else {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}
__device__ __forceinline__ uint32_t dc_map(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t dc_u32(const void* p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(dc_map(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 dc_u64(const void* p, int rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(dc_map(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint4 dc_u32x4(const void* p, int rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(dc_map(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float dc_f32(const void* p, int rank) { return __uint_as_float(dc_u32(p, rank)); }

// A value of every CTA, one per lane, put together (lane c and those eight apart read CTA c's).
template <typename V, class Read, class Op>
__device__ __forceinline__ V dc_over(int S, V none, Read&& read, Op&& op) {
    const int c = threadIdx.x & (kDcMaxCtas - 1);
    V v = none;
    if (c < S) v = read(c);
#pragma unroll
    for (int o = kDcMaxCtas / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <typename T>
struct DcVec {
    static constexpr int n = 16 / (int)sizeof(T);
};
__device__ __forceinline__ void dc_unpack(const uint4& v, float (&f)[4], const float*) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void dc_unpack(const uint4& v, float (&f)[8], const __half*) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ void dc_unpack(const uint4& v, float (&f)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t dc_lowest(const float*) { return 0xFF800000u; }
__device__ __forceinline__ uint32_t dc_lowest(const __half*) { return 0xFC00FC00u; }
__device__ __forceinline__ uint32_t dc_lowest(const __nv_bfloat16*) { return 0xFF80FF80u; }

// f(logit, place) for the logits of this warp's stretch of the slice
template <typename T, class F>
__device__ __forceinline__ void dc_scan(const T* slice, int seg, int warp, int lane, F&& f) {
    constexpr int N = DcVec<T>::n;
#pragma unroll 2
    for (int o = lane * N; o < seg; o += 32 * N) {
        float v[N];
        dc_unpack(*reinterpret_cast<const uint4*>(slice + warp * seg + o), v, (const T*)nullptr);
#pragma unroll
        for (int e = 0; e < N; ++e) f(v[e], warp * seg + o + e);
    }
}
__device__ __forceinline__ u64 dc_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the CTA of the values before this thread's, and over all.
__device__ __forceinline__ u64 dc_before(u64 v, u64* wsum, u64& all) {
    u64 incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
        if ((int)(threadIdx.x & 31) >= o) incl += t;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) wsum[threadIdx.x >> 5] = incl;
    __syncthreads();
    u64 base = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < kDwWarps; ++i) {
        const u64 t = wsum[i];
        if (i < (int)(threadIdx.x >> 5)) base += t;
        all += t;
    }
    return base + incl - v;
}
// keys[0 .. n) in falling order; n a power of two from 32 to 1024
__device__ __forceinline__ void dc_sort(u64* keys, int n) {
    const int tid = threadIdx.x;
#pragma unroll 1
    for (int k = 2; k <= n; k <<= 1)
#pragma unroll 1
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (tid < n / 2) {
                const int a = 2 * tid - (tid & (j - 1)), b = a + j;
                const u64 va = keys[a], vb = keys[b];
                if ((a & k) == 0 ? va < vb : va > vb) {
                    keys[a] = vb;
                    keys[b] = va;
                }
            }
            if (j > 32 || (j == 1 && k >= 64))  // (pairs up to 32 apart stay within a warp's 64 entries)
                __syncthreads();
            else
                __syncwarp();
        }
    __syncthreads();
}
__device__ __forceinline__ float dc_next(float v, bool up) {
    const uint32_t b = __float_as_uint(v);
    if (v == 0.f) return __uint_as_float(up ? 1u : 0x80000001u);
    return __uint_as_float((v > 0.f) == up ? b + 1 : b - 1);
}
// The least logit with y >= ymin.
__device__ __forceinline__ float dc_threshold(const DwRow& r, double ymin) {
    const float lowest = -3.402823466e38f;
    float t = (float)(r.mxd + ymin / r.c);
    t = t >= lowest ? fminf(t, r.mx) : lowest;  // (the quotient is not a number where T is infinite)
#pragma unroll 1
    for (int i = 0; i < 4 && !(dw_y(r, t) >= ymin) && t < r.mx; ++i) t = dc_next(t, true);
#pragma unroll 1
    for (int i = 0; i < 4 && t > lowest; ++i) {
        const float d = dc_next(t, false);
        if (!(dw_y(r, d) >= ymin)) break;
        t = d;
    }
    return t;
}

template <typename T>
struct DcRow {
    const DrawArgs& A;
    DcShared& sh;
    T* slice;
    DwRow r;
    int row, S, rank, n_slice, seg, off, warp, lane, tid;
    float floor_l, min_l;  // least logits with a weight, and that min-p keeps

    __device__ __forceinline__ uint32_t index_of(int c, int place) const { return (uint32_t)(c * n_slice + place - off); }
    __device__ __forceinline__ u64 weight(float l) const { return l >= floor_l ? dw_fixed(dw_y(r, l), r.F, sh.tab) : 0ull; }

    // Row to shared memory; this thread's largest logit.
    __device__ __forceinline__ float load(bool& nan) {
        constexpr int N = DcVec<T>::n;
        const T* lg = reinterpret_cast<const T*>(A.logits) + (size_t)row * A.ld;
        off = (int)((reinterpret_cast<uintptr_t>(lg) & 15) / sizeof(T));  // places count from the 16 bytes that the row starts in
        float tm = -INFINITY;
#pragma unroll 4
        for (int o = lane * N; o < seg; o += 32 * N) {
            const int place = warp * seg + o, i = rank * n_slice + place - off;
            uint4 v;
            if (i >= 0 && i + N <= A.V) {
                v = __ldcs(reinterpret_cast<const uint4*>(lg + i));
            } else {
                const uint32_t none = dc_lowest((const T*)nullptr);
                v = make_uint4(none, none, none, none);
                if (i + N > 0 && i < A.V) {
                    alignas(16) T part[N];
                    *reinterpret_cast<uint4*>(part) = v;
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (i + e >= 0 && i + e < A.V) part[e] = lg[i + e];
                    v = *reinterpret_cast<uint4*>(part);
                }
            }
            float f[N];
            dc_unpack(v, f, (const T*)nullptr);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                nan |= f[e] != f[e];
                tm = fmaxf(tm, f[e]);
            }
            *reinterpret_cast<uint4*>(slice + place) = v;
        }
        return tm;
    }

    // Lower bounds of the row's k-th largest logit from the threads' maxima: sh.thr_all, sh.thr_part (-inf: none).
    __device__ __forceinline__ void bounds(float tm, float mx, float mn, int k) {
        const int part = (k + S - 1) / S;
        const float s = mx > mn ? 255.0f / (mx - mn) : 0.f;
        int bin = 255;
        if (tm > -INFINITY) {
            bin = max(0, min(255, (int)((mx - tm) * s)));
            atomicAdd(&sh.tmhist[bin], 1u);
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += c[i] = sh.tmhist[lane * 8 + i];
            uint32_t incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            uint32_t at = incl - sum;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (at < (uint32_t)k && at + c[i] >= (uint32_t)k) sh.cross_all = lane * 8 + i;
                if (at < (uint32_t)part && at + c[i] >= (uint32_t)part) sh.cross_part = lane * 8 + i;
                at += c[i];
            }
        }
        __syncthreads();
        if (tm > -INFINITY) {
            const uint32_t key = dw_key(tm);
            if (bin <= sh.cross_all) atomicMin(&sh.key_all, key);
            if (bin <= sh.cross_part) atomicMin(&sh.key_part, key);
        }
        __syncthreads();
        if (tid == 0) {
            sh.thr_all = sh.key_all != ~0u ? dw_value(sh.key_all) : -INFINITY;
            sh.thr_part = sh.key_part != ~0u ? dw_value(sh.key_part) : -INFINITY;
        }
    }

    __device__ __forceinline__ void collect(float l, int place) {
        const int at = atomicAdd(&sh.n_list, 1);
        if (at < kDcList) sh.list[at] = (u64)dw_key(l) << 32 | (uint32_t)~index_of(rank, place);
    }
    // Entries in all CTAs' collections, more than kDcList where one of them ran over.
    __device__ __forceinline__ int collected() const {
        return dc_over(S, 0, [&](int c) { return min((int)dc_u32(&sh.n_list, c), kDcList + 1); }, [](int x, int y) { return x + y; });
    }
    __device__ __forceinline__ u64 over_ctas(const u64* p) const {
        return dc_over(S, (u64)0, [&](int c) { return dc_u64(p, c); }, [](u64 x, u64 y) { return x + y; });
    }
    // All collections, sorted, to sh.keys.  (Every thread holds entries 2 tid and 2 tid + 1 from here on.)
    __device__ __forceinline__ void merge(int n, u64 (&key)[2]) {
        int np = 32, at = 0;
        while (np < n) np <<= 1;
#pragma unroll 1
        for (int c = 0; c < S; ++c) {
            const int nc = (int)dc_u32(&sh.n_list, c);
            for (int i = tid; i < nc; i += kDwThreads) sh.keys[at + i] = dc_u64(&sh.list[i], c);
            at += nc;
        }
        for (int i = n + tid; i < np; i += kDwThreads) sh.keys[i] = 0;
        __syncthreads();
        dc_sort(sh.keys, np);
#pragma unroll
        for (int e = 0; e < 2; ++e) key[e] = 2 * tid + e < n ? sh.keys[2 * tid + e] : 0ull;
    }
    // Of the sorted entries those that come before number `most` and before which, with `above` before the first, the weight is under `share` of all that
    // `most` leaves (share <= 0: no such limit; total 0: the sum up to here): how many, their weights, and the sum up to the last of `most`.
    __device__ __forceinline__ int cut_of(const u64 (&key)[2], int n, int most, u64 above, float share, u64 total, u64 (&w)[2], u64& P, u64& sum) {
        u64 all, before;
#pragma unroll
        for (int e = 0; e < 2; ++e) w[e] = 2 * tid + e < min(n, most) ? weight(dw_value((uint32_t)(key[e] >> 32))) : 0ull;
        before = above + dc_before(w[0] + w[1], sh.wsum, all);
        sum = above + all;
        P = share > 0.f ? dw_share(share, total ? total : sum) : ~0ull;
        const int k0 = w[0] && before < P, k1 = w[1] && before + w[0] < P;
        if (!k0) w[0] = 0;
        if (!k1) w[1] = 0;
        return __syncthreads_count(k0) + __syncthreads_count(k1);
    }

    // The draw among collected entries alone (one CTA): entry e of the thread is kept where its weight is not 0.
    __device__ __forceinline__ void draw_list(const u64 (&key)[2], u64 (&w)[2], int kept) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (w[e] && !(dw_value((uint32_t)(key[e] >> 32)) >= min_l)) w[e] = 0;
        u64 total, unused = dc_before(w[0] + w[1], sh.wsum, total);
        (void)unused;
        const u64 U = dw_target(A.u[row], total);
        u64* ws = sh.list;  // (all collections have been read)
        if (kept <= 128) {
            // running sums in vocabulary order by comparing indices
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * tid + e < kept) ws[2 * tid + e] = w[e];
            __syncthreads();
            if (tid < kept) {
                const u64 mine = sh.keys[tid];
                const uint32_t inv = (uint32_t)mine;
                u64 before = 0;
                for (int j = 0; j < kept; ++j)
                    if ((uint32_t)sh.keys[j] > inv) before += ws[j];
                if (ws[tid] && before <= U && before + ws[tid] > U) dw_result(A, row, ~inv, dw_logprob(r, dw_value((uint32_t)(mine >> 32)), total));
            }
            return;
        }
        // sorted by their index (as ~index << 32 | place, rising index = falling word), then a prefix sum
        __syncthreads();
        int np = 32;
        while (np < kept) np <<= 1;
        for (int i = tid; i < np; i += kDwThreads) ws[i] = i < kept ? (u64)(uint32_t)sh.keys[i] << 32 | (uint32_t)i : 0ull;
        __syncthreads();
        dc_sort(ws, np);
        u64 v[2], k2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 2 * tid + e;
            k2[e] = i < kept ? sh.keys[(uint32_t)ws[i]] : 0ull;
            const float l = dw_value((uint32_t)(k2[e] >> 32));
            v[e] = i < kept && l >= min_l ? weight(l) : 0ull;
        }
        u64 all, before = dc_before(v[0] + v[1], sh.wsum, all);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (v[e] && before <= U && before + v[e] > U) dw_result(A, row, ~(uint32_t)k2[e], dw_logprob(r, dw_value((uint32_t)(k2[e] >> 32)), total));
            before += v[e];
        }
    }

    // The draw among all logits down to `cut` (key << 32 | ~index) and min_l, from the warps' sums in sh.seg of all CTAs and the `kept` entries of a region.
    __device__ __forceinline__ void draw_segments(u64 cut, int kept) {
        const int n = S * kDwWarps;
        __syncthreads();
        if (tid < n) sh.segs[tid] = dc_u64(&sh.seg[tid % kDwWarps], tid / kDwWarps);
        __syncthreads();
        for (int i = tid; i < kept; i += kDwThreads) {
            const u64 k = sh.keys[i];
            const float l = dw_value((uint32_t)(k >> 32));
            const int place = (int)~(uint32_t)k + off;
            if (l >= min_l) atomicAdd(&sh.segs[place / n_slice * kDwWarps + place % n_slice / seg], weight(l));
        }
        __syncthreads();
        u64 total, w = tid < n ? sh.segs[tid] : 0ull;
        const u64 before = dc_before(w, sh.wsum, total);
        const u64 U = dw_target(A.u[row], total);
        if (w && before <= U && before + w > U) {
            sh.found = tid;
            sh.segs[0] = before;
        }
        __syncthreads();
        const int f = sh.found;
        if (f / kDwWarps != rank) return;
        // that stretch again: consecutive logits per thread
        const u64 base = sh.segs[0];
        const int from = part_of(f, tid), to = part_of(f, tid + 1);
        u64 sum = 0;
        for (int i = from; i < to; ++i) sum += kept_weight(i, cut);
        u64 all, b = base + dc_before(sum, sh.wsum, all);
        if (sum && b <= U && b + sum > U)
            for (int i = from; i < to; ++i) {
                b += kept_weight(i, cut);
                if (b > U) {
                    dw_result(A, row, index_of(rank, i), dw_logprob(r, dw_f32(slice[i]), total));
                    break;
                }
            }
    }
    __device__ __forceinline__ int part_of(int f, int t) const { return f % kDwWarps * seg + (int)((unsigned)seg * (unsigned)t / (unsigned)kDwThreads); }
    __device__ __forceinline__ u64 kept_weight(int place, u64 cut) const {
        const float l = dw_f32(slice[place]);
        if (!(l >= min_l)) return 0;
        return ((u64)dw_key(l) << 32 | (uint32_t)~index_of(rank, place)) >= cut ? weight(l) : 0ull;
    }
};

template <typename T>
__global__ void __launch_bounds__(kDwThreads, 2) draw_cluster_kernel(DrawArgs A, int S, int n_slice) {
    extern __shared__ __align__(16) unsigned char dc_smem[];
    DcShared& sh = *reinterpret_cast<DcShared*>(dc_smem);
    DcRow<T> R = {A, sh, reinterpret_cast<T*>(dc_smem + sizeof(DcShared))};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    R.tid = tid, R.lane = lane, R.warp = warp;
    R.S = S;
    R.rank = S > 1 ? (int)dc_rank() : 0;
    R.row = (int)blockIdx.x / S;
    R.n_slice = n_slice;
    R.seg = n_slice / kDwWarps;
    R.r = dw_row(A, R.row);
    DwRow& r = R.r;
    dw_fill_table(sh.tab);
    const bool small = A.V <= kDcList;
    const bool list_k = !r.greedy && !small && r.top_k && r.top_k <= (uint32_t)kDcFastK, list_p = !r.greedy && !small && !r.top_k && r.top_p > 0.f;
    const bool list = !r.greedy && (small || list_k || list_p);
    bool binned = !r.greedy && !list && r.top_k;

    // ---- the row, its largest logit, bounds of what is kept
    for (int i = tid; i < kDcBins; i += kDwThreads) sh.hist[i] = 0u;
    if (tid < 256) sh.tmhist[tid] = 0u;
    if (tid == 0) {
        sh.n_list = 0;
        sh.n_above = 0;
        sh.key_all = sh.key_part = ~0u;
        sh.cross_all = sh.cross_part = -1;
        sh.thr_all = sh.thr_part = -INFINITY;
        sh.first = kDwNone;
        sh.total = sh.mass = 0;
    }
    bool nan = false;
    const float tm = R.load(nan);
    float mx = tm, mn = tm > -INFINITY ? tm : INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0) sh.red[warp] = mx, sh.redmin[warp] = mn;
    nan = __syncthreads_or(nan);
#pragma unroll
    for (int i = 0; i < kDwWarps; ++i) mx = fmaxf(mx, sh.red[i]), mn = fminf(mn, sh.redmin[i]);
    if (tid == 0) sh.mx = mx, sh.nan = nan;
    if (list_k || list_p) R.bounds(tm, mx, mn, list_k ? (int)r.top_k : kDcTryK);
    dc_sync(S);
    const float mine = mx;
    const auto larger = [](float x, float y) { return fmaxf(x, y); };
    mx = dc_over(S, -INFINITY, [&](int c) { return dc_f32(&sh.mx, c); }, larger);
    nan = dc_over(S, 0u, [&](int c) { return dc_u32(&sh.nan, c); }, [](uint32_t x, uint32_t y) { return x | y; }) != 0u;
    const int owner = dc_over(S, S, [&](int c) { return dc_f32(&sh.mx, c) == mx ? c : S; }, [](int x, int y) { return min(x, y); });  // the first CTA with the largest logit
    const float thr_all = dc_over(S, -INFINITY, [&](int c) { return dc_f32(&sh.thr_all, c); }, larger);
    const float thr_part = dc_over(S, INFINITY, [&](int c) { return dc_f32(&sh.thr_part, c); }, [](float x, float y) { return fminf(x, y); });
    if (nan || mx == -INFINITY || r.greedy) {
        if (nan || mx == -INFINITY) {
            if (R.rank == 0 && tid == 0) dw_result(A, R.row, kDwNone, nan ? NAN : -INFINITY);
        } else if (R.rank == owner && mine == mx) {
            uint32_t best = kDwNone;
            dc_scan<T>(R.slice, R.seg, warp, lane, [&](float l, int place) {
                if (l == mx) best = min(best, (uint32_t)place);
            });
            best = __reduce_min_sync(0xffffffffu, best);
            if (lane == 0) atomicMin(&sh.first, best);
            __syncthreads();
            if (tid == 0) dw_result(A, R.row, R.index_of(R.rank, (int)sh.first), 0.f);
        }
        dc_sync(S);
        return;
    }
    r.mx = mx;
    r.mxd = (double)mx;
    R.floor_l = dc_threshold(r, -40.0);
    R.min_l = r.ymin > -40.0 ? dc_threshold(r, r.ymin) : R.floor_l;

    bool plain = false;  // left to radix passes
    u64 total = 0;       // weight of the whole row, where top-p needs it
    if (list) {
        const float thr = fmaxf(fmaxf(thr_all, thr_part), -3.402823466e38f);  // (-inf is never drawn)
        u64 sum = 0, mass = 0;
        dc_scan<T>(R.slice, R.seg, warp, lane, [&](float l, int place) {
            if (l >= thr) R.collect(l, place);
            if (list_p && l >= R.floor_l) {
                const u64 w = dw_fixed(dw_y(r, l), r.F, sh.tab);
                sum += w;
                if (l >= thr) mass += w;
            }
        });
        if (list_p) {
            sum = dc_warp_sum(sum);
            mass = dc_warp_sum(mass);
            if (lane == 0) atomicAdd(&sh.total, sum), atomicAdd(&sh.mass, mass);
        }
        dc_sync(S);
        const int n = R.collected();
        bool here = n <= kDcList;
        if (list_p) {
            total = R.over_ctas(&sh.total);
            here = here && R.over_ctas(&sh.mass) >= dw_share(r.top_p, total);
            binned = !here;
        } else {
            plain = !here;
        }
        if (here) {
            if (R.rank == 0) {
                u64 key[2], w[2], P, sum;
                R.merge(n, key);
                const int kept = R.cut_of(key, n, r.top_k ? (int)r.top_k : n, 0, r.top_p, total, w, P, sum);
                R.draw_list(key, w, kept);
            }
            dc_sync(S);
            return;
        }
    }
    u64 cut = 0;
    int kept = 0;
    bool summed = false;  // sh.seg holds the sums of what lies above the region of the cut
    if (binned) {
        // ---- histogram of the distance to the maximum
        const float s = fminf(((float)kDcBins - 0.5f) / fminf((float)(40.0 / r.c), 3e38f), 1e30f);  // (what has a weight is in a bin)
        const auto where = [&](float l) { return fmaxf(mx - l, 0.f) * s; };                           // (0 for inf - inf)
        dc_scan<T>(R.slice, R.seg, warp, lane, [&](float l, int) {
            const float q = where(l);
            if (q < (float)kDcBins) atomicAdd(&sh.hist[(int)q], 1u);
        });
        dc_sync(S);
        uint32_t cnt[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kDcMaxCtas; ++c)
            if (c < S) {
                const uint4 h = dc_u32x4(&sh.hist[4 * tid], c);
                cnt[0] += h.x, cnt[1] += h.y, cnt[2] += h.z, cnt[3] += h.w;
            }
        // counts and (nearly) weights before this thread's bins
        u64 all_cnt;
        const u64 cnt_before = dc_before(cnt[0] + cnt[1] + cnt[2] + cnt[3], sh.wsum, all_cnt);
        const float step = -40.0f / ((float)kDcBins - 0.5f);
        u64 near[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) near[i] = (u64)((float)cnt[i] * exp2f(((float)(4 * tid + i) + 0.5f) * step) * 16777216.0f);
        u64 near_all;
        const u64 near_before = dc_before(near[0] + near[1] + near[2] + near[3], sh.wsum, near_all);
        // One collection: logits of bins b1 .. b2, the weight and number of those before them.
        auto region = [&](int b1, int b2, u64& above, int& n_above) {
            const float q1 = (float)b1, q2 = (float)(b2 + 1);
            u64 sum = 0;
            int na = 0;
            dc_scan<T>(R.slice, R.seg, warp, lane, [&](float l, int place) {
                const float q = where(l);
                if (q < q1) {
                    ++na;
                    sum += R.weight(l);
                } else if (q < q2) {
                    R.collect(l, place);
                }
            });
            sum = dc_warp_sum(sum);
            na = __reduce_add_sync(0xffffffffu, na);
            if (lane == 0) {
                sh.seg[warp] = sum;
                atomicAdd(&sh.n_above, na);
            }
            dc_sync(S);
            n_above = dc_over(S, 0, [&](int c) { return (int)dc_u32(&sh.n_above, c); }, [](int x, int y) { return x + y; });
            (void)dc_before(tid < S * kDwWarps ? dc_u64(&sh.seg[tid % kDwWarps], tid / kDwWarps) : 0ull, sh.wsum, above);
        };
        auto find_bin = [&](u64 before, const auto (&v)[4], u64 want) {  // the bin where the running sum reaches `want`
            __syncthreads();
            if (tid == 0) sh.bin = kDcBins - 1;
            __syncthreads();
            u64 at = before;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (at < want && at + v[i] >= want) sh.bin = 4 * tid + i;
                at += v[i];
            }
            __syncthreads();
            return sh.bin;
        };
        u64 above = 0, key[2] = {0, 0}, w[2], P = ~0ull, sum;
        int n_above = 0, n = 0, b1 = 0;
        bool p_left = r.top_p > 0.f;
        if (r.top_k && all_cnt > r.top_k) {
            b1 = find_bin(cnt_before, cnt, r.top_k);
            region(b1, b1, above, n_above);
            n = R.collected();
            plain = n > kDcList;
            if (!plain) {
                R.merge(n, key);
                kept = R.cut_of(key, n, (int)r.top_k - n_above, above, r.top_p, 0, w, P, total);
                p_left = p_left && above >= P;  // top-p's cut lies further up
            }
        } else if (r.top_k && p_left) {  // top-k keeps all that have a weight
            region(kDcBins, kDcBins, total, n_above);
        }
        if (p_left && !plain) {
            P = dw_share(r.top_p, total);
            const u64 want = (u64)((double)P * exp2(24.0 - (double)r.F));  // in the units of `near`
            const int b = find_bin(near_before, near, want > 0 ? want : 1);
            if (r.top_k) dc_sync(S);  // (the collection before this one may still be read)
            if (tid == 0) sh.n_list = sh.n_above = 0;
            __syncthreads();
            b1 = max(b - 1, 0);
            region(b1, b + 1, above, n_above);
            n = R.collected();
            plain = n > kDcList || above >= P;
            if (!plain) {
                R.merge(n, key);
                kept = R.cut_of(key, n, n, above, r.top_p, total, w, P, sum);
                plain = sum < P;  // the cut lies further down
            }
        }
        if (!plain && kept > 0) {
            cut = sh.keys[kept - 1];
            summed = !(where(R.min_l) < (float)b1);  // min-p keeps all that lies above the region
            if (!summed) kept = 0;
        }
    }
    if (plain) {
        if (R.rank == 0) dw_row_plain<T>(A, R.row, *reinterpret_cast<DwPlainShared*>(R.slice));
        dc_sync(S);
        return;
    }
    if (!summed) {
        // min-p's cut is the stricter one, or there is no other
        u64 sum = 0;
        dc_scan<T>(R.slice, R.seg, warp, lane, [&](float l, int) {
            if (l >= R.min_l) sum += dw_fixed(dw_y(r, l), r.F, sh.tab);
        });
        sum = dc_warp_sum(sum);
        if (binned) dc_sync(S);  // (the sums of a region may still be read)
        if (lane == 0) sh.seg[warp] = sum;
        dc_sync(S);
        cut = 0;
        kept = 0;
    }
    R.draw_segments(cut, kept);
    dc_sync(S);  // no CTA leaves while its shared memory may be read
}

}  // namespace rsv
