// Drawing with a row held in the shared memory of a cluster of CTAs (draw.cuh has the definition and the arithmetic).
//
// The logits are read from global memory once, with their maximum; everything else works on shared memory.  The cut that top-k and top-p make is
// found without sorting the row:
//   list    Every thread keeps the largest of its own logits.  The k-th largest of a CTA's 256 such maxima is a lower bound of the row's k-th largest
//           logit, and so is the smallest over the CTAs of the (k / CTAs)-th; the logits from the larger of the two on are collected (k and a few more) and
//           sorted by value and index, and the cut lies among them.  With top-p and no top-k the 128 largest are tried: their weight tells whether
//           the cut lies among them.
//   region  Otherwise the cut lies in a stretch of values known from the pass that summed the weights (three stretches, divided by bounds from the threads'
//           maxima).  A histogram of that stretch in 512 linear bins says near which bin the cut is; the logits of that bin and its neighbours are
//           collected and sorted, the weight of all larger ones is summed exactly, and the sums tell whether the cut is there.
//   zoom    Bins with more than 384 logits (a flat row, a large vocabulary, 16-bit logits) are divided into 512 bins again, up to four times; of equal logits
//           as many are kept as the weight left, or the number, needs.  74 rows of 131072 logits with a deviation of 0.3 and top-p 0.9: 0.16 ms, where one
//           CTA a row took 2.1 ms; 80 rows of 65536 bf16 logits with seven values: 0.12 ms and 3.2 ms.
//   neither Where more than 384 logits are equal to a small top-k's last, or four divisions were not enough, one CTA does the row by radix passes
//           (dw_row_plain).
// Without top-k and top-p no cut is needed: min-p's is a value that follows from the maximum.
//
// The draw: sums of the kept weights per warp, whose logits follow each other in the vocabulary, then the one warp's stretch again, split over a CTA.
//
// What the CTAs tell each other is written into the receiver's shared memory before a cluster barrier, so that nobody has to stay for others to read: one
// CTA finishes a row while the others' places go to the next rows.
//
// Rows of 65536 fp32 logits, us on the GPU: one row 4.7 (greedy), 10.5 (top-k 50, top-p 0.9), 24 (top-p 0.9), bound by barriers and one CTA's chain; 1024 rows 78 (3.4 TB/s),
// 129 and 432, bound by instructions.  Five CTAs of 48 registers on an SM.
#pragma once
#include "draw.cuh"
#include "tc_ptx.cuh"

namespace rsv {

constexpr int kDcList = 384;  // entries of a collection
constexpr int kDcPer = 2;     // at most, of a thread
constexpr int kDcBins = 512;
constexpr int kDcBinsPer = kDcBins / kDwThreads;
static_assert(kDcBinsPer == 2, "bins are read in pairs");
constexpr int kDcFastK = 160;                   // most entries of top-k that are collected whole
constexpr int kDcMostPart = kDwThreads * 7 / 8;  // most of a CTA's thread maxima that are asked for
constexpr int kDcTryK = 128;                     // entries tried for top-p alone,
constexpr int kDcTryPart = kDwThreads * 3 / 8;   // and of one CTA's thread maxima
constexpr int kDcMaxCtas = 8;
constexpr int kDcZooms = 4;   // times that bins are divided again
constexpr int kDcMarked = 8;  // vectors a thread can mark the logits of
static_assert(kDcMaxCtas * kDwWarps == 64 && kDwWarps == 8, "two stretches a lane; warps add up among eight lanes");
constexpr int kDcSliceBytes = 32 * 1024;  // a CTA's part of a row, as long as eight CTAs suffice
constexpr int kDcMostSliceBytes = 192 * 1024;

struct DcSums {
    u64 total, n, from_a, from_c;  // weight of the slice, entries collected, weights from the two bounds on
};
struct DcZoom {  // what a cut in bins with too many logits goes on from
    float mx, mn, from_l, to_l;
    const u64* base;
    u64 base_all, total;
};
struct DcShared {
    // written by the other CTAs
    float4 top[kDcMaxCtas];  // largest logit (NaN: there is one), smallest of the threads' maxima, two lower bounds
    DcSums sums[kDcMaxCtas];
    u64 segs[kDcMaxCtas * kDwWarps];  // weights of the warps' stretches
    int above[kDcMaxCtas];            // logits above a region
    int ties[kDcMaxCtas * kDwWarps];  // and in it, of the warps' stretches
    u64 left, cut_p;                  // what top-k leaves; 0: the row is done
    int n_list[3];                    // entries of the collections below (one after the other)
    alignas(16) u64 list[kDcList];    // key << 32 | ~index
    // read by the other CTAs
    alignas(16) uint2 hist[kDcBins];  // logits of a bin, and their weights relative to that of its upper end
    // this CTA's own
    union {
        alignas(16) u64 mine[kDcList];
        alignas(16) uint32_t tmhist[256];  // (before anything is collected)
    };
    double tab[16], rate, least;
    u64 wsum[kDwWarps], seg_a[kDwWarps], seg_c[kDwWarps], before, target, sum;
    float red[kDwWarps], redmin[kDwWarps], thr_all, thr_part, floor_l, min_l;
    uint32_t first;
    int n_mine, n_above[kDwWarps], bin, bin_to, n_in, found;
    DcZoom zoom;
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
// The two halves of a barrier: a CTA's shared memory may be written to once it has begun.
__device__ __forceinline__ void dc_arrive(int S) {
    if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void dc_wait(int S) {
    if (S > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}
__device__ __forceinline__ uint32_t dc_map(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint4 dc_u32x4(const void* p, int rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(dc_map(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void dc_put(int rank, int* p, int v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dc_map(p, rank)), "r"(v) : "memory"); }
__device__ __forceinline__ void dc_put(int rank, u64* p, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dc_map(p, rank)), "l"(v) : "memory"); }
__device__ __forceinline__ void dc_put(int rank, float4* p, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dc_map(p, rank)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ int dc_add(int rank, int* p, int v) {
    int before;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(before) : "r"(dc_map(p, rank)), "r"(v) : "memory");
    return before;
}
// Largest of three (NaN where one is), and largest and smallest of a warp's.
__device__ __forceinline__ float dc_max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float dc_warp_max(float v) {
    float d;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}
__device__ __forceinline__ float dc_warp_min(float v) {
    float d;
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}
// A value of every CTA, one per lane (lane c and those eight apart have CTA c's), put together.
template <typename V, class Op>
__device__ __forceinline__ V dc_all(V v, Op&& op) {
#pragma unroll
    for (int o = kDcMaxCtas / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
struct DcAdd {
    __device__ __forceinline__ u64 operator()(u64 x, u64 y) const { return x + y; }
    __device__ __forceinline__ int operator()(int x, int y) const { return x + y; }
};

template <int N>
__device__ __forceinline__ float dc_largest(const float (&v)[N]) {
    float m = dc_max3(v[0], v[1], v[2]);
#pragma unroll
    for (int e = 3; e + 1 < N; e += 2) m = dc_max3(m, v[e], v[e + 1]);
    return fmaxf(m, v[N - 1]);
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

// Sum over the warp of values under 2^52, in two halves.
__device__ __forceinline__ u64 dc_warp_sum(u64 v) {
    return ((u64)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26)) << 26) + __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3FFFFFFu);
}
// Sum over the CTA of the values before this thread's, and over all.  (A function of its own, as the sort: the code of a row is run once, and has to be fetched.)
__device__ __noinline__ ulonglong2 dc_before2(u64 v, u64* wsum) {
    u64 incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
        if ((int)(threadIdx.x & 31) >= o) incl += t;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) wsum[threadIdx.x >> 5] = incl;
    __syncthreads();
    u64 base = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kDwWarps; ++i) {
        const u64 t = wsum[i];
        if (i < (int)(threadIdx.x >> 5)) base += t;
        sum += t;
    }
    return make_ulonglong2(base + incl - v, sum);
}
__device__ __forceinline__ u64 dc_before(u64 v, u64* wsum, u64& all) {
    const ulonglong2 t = dc_before2(v, wsum);
    all = t.y;
    return t.x;
}
// keys[0 .. n) in falling order, all different: a key's place is the number of larger ones.
__device__ __noinline__ void dc_sort(u64* keys, int n) {
    const int tid = threadIdx.x;
    u64 mine[kDcPer];
    int place[kDcPer];
#pragma unroll
    for (int e = 0; e < kDcPer; ++e) mine[e] = tid + e * kDwThreads < n ? keys[tid + e * kDwThreads] : ~0ull, place[e] = 0;
    if (tid == 0 && n < kDcList) keys[n] = 0;  // (pairs are read)
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kDcPer; ++e)
        if (tid + e * kDwThreads < n)
#pragma unroll 4
            for (int j = 0; j < n; j += 2) {
                const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(&keys[j]);
                place[e] += (k.x > mine[e]) + (k.y > mine[e]);
            }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kDcPer; ++e)
        if (tid + e * kDwThreads < n) keys[place[e]] = mine[e];
    __syncthreads();
}
// The least logit l (lowest finite .. max) with (l - max) c >= ymin, by a half warp: the quotient, and sixteen floats around it.
__device__ __forceinline__ float dc_threshold(const DwRow& r, double ymin) {
    const float lowest = -3.402823466e38f;
    float t = (float)(r.mxd + ymin * (double)r.T * 0.69314718055994531);
    t = t >= lowest ? fminf(t, r.mx) : lowest;
    const uint32_t b = __float_as_uint(t);
    int at = b & 0x80000000u ? (int)(0x80000000u - b) : (int)b;  // floats in order, +0 and -0 the same
    at += (int)(threadIdx.x & 15) - 8;
    const float v = at < 0 ? __uint_as_float(0x80000000u - (uint32_t)at) : __uint_as_float((uint32_t)at);
    const bool ok = v <= r.mx && v >= lowest && dw_y(r, v) >= ymin;
    const uint32_t half = (__ballot_sync(0xffffffffu, ok) >> (threadIdx.x & 16)) & 0xFFFFu;
    return half ? __shfl_sync(0xffffffffu, v, (threadIdx.x & 16) + __ffs(half) - 1) : t;
}

// How a row is finished: not by this CTA, by min-p's cut, by the cut in `cut`, by radix passes.
enum DcEnd { kDcDone, kDcByMinP, kDcByCut, kDcByPasses };
struct DcCut {
    u64 cut, limit;  // key << 32 | ~index of the last kept; by min-p: with more weight than the limit top-p's cut is further up after all
    int kept;        // listed entries that are kept
};

template <typename T>
struct DcRow {
    const DrawArgs& A;
    DcShared& sh;
    T* slice;
    DwRow r;
    int row, S, rank, n_slice, seg, off, warp, lane, tid;
    float floor_l, min_l;  // least logits with a weight, and that min-p keeps
    static constexpr int N = DcVec<T>::n;

    __device__ __forceinline__ uint32_t index_of(int place) const { return (uint32_t)(rank * n_slice + place - off); }
    __device__ __forceinline__ u64 weight(float l) const { return l >= floor_l ? dw_fixed(r, l, sh.tab) : 0ull; }
    __device__ __forceinline__ u64 weight_of(u64 key) const { return weight(dw_value((uint32_t)(key >> 32))); }

    // f(vector, its largest logit, place of its first, its number) for this warp's stretch of the slice, whose vectors are as many for all lanes
    template <class F>
    __device__ __forceinline__ void scan(F&& f) const {
        int i = 0;
#pragma unroll 1
        for (int o = lane * N; o < seg; o += 32 * N) {
            float v[N];
            dc_unpack(*reinterpret_cast<const uint4*>(slice + warp * seg + o), v, (const T*)nullptr);
            f(v, dc_largest(v), warp * seg + o, i++);
        }
    }
    // The marks of a vector's logits from `least` on (bit 4 i + e: logit e of a group of four of vector i).
    __device__ __forceinline__ void mark(uint32_t (&marks)[N / 4], const float (&v)[N], int i, float least) const {
#pragma unroll
        for (int g = 0; g < N / 4; ++g) {
            uint32_t s[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) asm("set.ge.u32.f32 %0, %1, %2;" : "=r"(s[e]) : "f"(v[4 * g + e]), "f"(least));
            marks[g] |= ((s[0] & 1u) | (s[1] & 2u) | (s[2] & 4u) | (s[3] & 8u)) << (4 * i);
        }
    }
    // f(four logits, their places) for the marked ones, or, where a stretch is too long for marks, for all; -inf where there are no more.  (Four at a time: one
    // after the other each would wait for the one before it.)
    template <class F>
    __device__ __forceinline__ void each(const uint32_t (&marks)[N / 4], F&& f) const {
        if (seg <= 32 * N * kDcMarked) {
#pragma unroll
            for (int g = 0; g < N / 4; ++g) {
                uint32_t m = marks[g];
                const int first = warp * seg + lane * N + 4 * g;
#pragma unroll 1
                while (__any_sync(0xffffffffu, m != 0u)) {
                    float l[4];
                    int at[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int b = m ? __ffs(m) - 1 : 0;
                        at[e] = first + (b >> 2) * 32 * N + (b & 3);
                        l[e] = m ? dw_f32(slice[at[e]]) : -INFINITY;
                        m &= m - 1;
                    }
                    f(l, at);
                }
            }
        } else {
#pragma unroll 1
            for (int o = 0; o < seg; o += 128) {
                float l[4];
                int at[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    at[e] = warp * seg + o + 32 * e + lane;  // (a stretch is a multiple of 128 logits)
                    l[e] = dw_f32(slice[at[e]]);
                }
                f(l, at);
            }
        }
    }
    // g(logit, weight) for all logits of the vectors where a lane's largest is from `least` on (weights of logits under floor_l are any number).  Four chains at
    // a time: branches around single ones would put them in a row.  The weights are whole numbers in fp64, and so are a thread's sums of them.
    template <class G>
    __device__ __forceinline__ void weights(const float (&v)[N], float largest, float least, G&& g) const {
        if (!__any_sync(0xffffffffu, largest >= least)) return;
#pragma unroll 1
        for (int q = 0; q < N; q += 4) {
            float l[4];
            double w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e] = N == 4 ? v[e] : q ? v[(e + 4) % N] : v[e];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = dw_whole(r, l[e], sh.tab);
#pragma unroll
            for (int e = 0; e < 4; ++e) g(l[e], w[e]);
        }
    }

    // Logits at `place` of the slice, -inf where the row has none.
    __device__ __forceinline__ uint4 fetch(const T* lg, int place) const {
        const int i = rank * n_slice + place - off;
        if (i >= 0 && i + N <= A.V) return __ldcs(reinterpret_cast<const uint4*>(lg + i));
        const uint32_t none = dc_lowest((const T*)nullptr);
        uint4 v = make_uint4(none, none, none, none);
        if (i + N > 0 && i < A.V) {
            T* part = slice + place;  // (put together where the vector goes)
            *reinterpret_cast<uint4*>(part) = v;
#pragma unroll 1
            for (int e = 0; e < N; ++e)
                if (i + e >= 0 && i + e < A.V) part[e] = lg[i + e];
            v = *reinterpret_cast<uint4*>(part);
        }
        return v;
    }
    // Row to shared memory; this thread's largest logit (NaN where there is one).  `meanwhile` runs while the first loads are on their way.
    template <class F>
    __device__ __forceinline__ float load(F&& meanwhile) {
        constexpr int B = 6;  // (8 need more registers than there are, and spill: 4.8 instead of 4.5 us for the largest logit of 65536)
        const T* lg = reinterpret_cast<const T*>(A.logits) + (size_t)row * A.ld;
        off = (int)((reinterpret_cast<uintptr_t>(lg) & 15) / sizeof(T));  // places count from the 16 bytes that the row starts in
        const bool whole = rank * n_slice >= off && (rank + 1) * n_slice - off <= A.V;
        const uint4* src = reinterpret_cast<const uint4*>(lg - off + (ptrdiff_t)rank * n_slice + warp * seg);  // (read where the slice is whole)
        float tm = -INFINITY;
#pragma unroll 1
        for (int o = lane * N; o < seg; o += 32 * N * B) {
            uint4 v[B];
            if (whole) {
#pragma unroll
                for (int b = 0; b < B; ++b)
                    if (o + 32 * N * b < seg) v[b] = __ldcs(src + o / N + 32 * b);
            } else {
#pragma unroll
                for (int b = 0; b < B; ++b)
                    if (o + 32 * N * b < seg) v[b] = fetch(lg, warp * seg + o + 32 * N * b);
            }
            if (o < 32 * N) meanwhile();
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (o + 32 * N * b < seg) {
                    float f[N];
                    dc_unpack(v[b], f, (const T*)nullptr);
#pragma unroll
                    for (int e = 0; e < N; e += 2) tm = dc_max3(tm, f[e], f[e + 1]);
                    *reinterpret_cast<uint4*>(slice + warp * seg + o + 32 * N * b) = v[b];
                }
        }
        return tm;
    }

    // Lower bounds of the row's k-th largest logit from the threads' maxima (-inf: none): the k-th of this CTA's, and its (k / CTAs)-th, found to within the
    // bins of a histogram; a hundredth of a bin is left for rounding (where that is not enough, too few are collected, which is seen).
    __device__ __forceinline__ void bounds(float tm, float mx, float mn, int k) {
        const int part = (k + S - 1) / S;
        const float s = mx > mn ? 255.0f / (mx - mn) : 0.f;
        if (tm > -INFINITY) atomicAdd(&sh.tmhist[max(0, min(255, (int)((mx - tm) * s)))], 1u);
        __syncthreads();
        if (warp == 0) {
            const uint4 h0 = reinterpret_cast<const uint4*>(sh.tmhist)[2 * lane], h1 = reinterpret_cast<const uint4*>(sh.tmhist)[2 * lane + 1];
            const uint32_t c[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
            uint32_t sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += c[i];
            uint32_t at = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, at, o);
                if (lane >= o) at += t;
            }
            at -= sum;
            const float width = (mx - mn) / 255.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float edge = mx > mn ? mx - ((float)(lane * 8 + i) + 1.01f) * width : mx;
                if (at < (uint32_t)k && at + c[i] >= (uint32_t)k) sh.thr_all = edge;
                if (at < (uint32_t)part && at + c[i] >= (uint32_t)part) sh.thr_part = edge;
                at += c[i];
            }
        }
        __syncthreads();
    }

    __device__ __forceinline__ void collect(float l, int place) {
        const int at = atomicAdd(&sh.n_mine, 1);
        if (at < kDcList) sh.mine[at] = (u64)dw_key(l) << 32 | (uint32_t)~index_of(place);
    }
    // This CTA's collection to the end of the first CTA's list number c, and its number back to none.  (Too many entries: the number says so.)
    __device__ __forceinline__ void hand_in(int c) {
        __syncthreads();
        const int n = sh.n_mine;
        if (tid == 0) sh.found = dc_add(0, &sh.n_list[c], n);
        __syncthreads();
        const int at = sh.found;
        if (tid == 0) sh.n_mine = 0;
#pragma unroll 1
        for (int i = tid; i < min(n, kDcList); i += kDwThreads)
            if (at + i < kDcList) dc_put(0, &sh.list[at + i], sh.mine[i]);
    }
    // Entries of a sorted list that a thread has: kDcPer consecutive ones, or one where they are no more than threads.
    __device__ __forceinline__ int entry(int n, int e) const { return n <= kDwThreads ? (e ? kDcList : tid) : kDcPer * tid + e; }
    __device__ __forceinline__ void sorted(int n, u64 (&key)[kDcPer]) {
        dc_sort(sh.list, n);
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) key[e] = entry(n, e) < n ? sh.list[entry(n, e)] : 0ull;
    }
    // Of the sorted entries those that come before number `most` and before which, with `above` before the first, the weight is under `share` of all that
    // `most` leaves (share <= 0: no such limit; total 0: the sum up to here): how many, their weights, and the sum up to the last of `most`.
    __device__ __forceinline__ int cut_of(const u64 (&key)[kDcPer], int n, int most, u64 above, float share, u64 total, u64 (&w)[kDcPer], u64& P, u64& sum) {
        u64 all, before, own = 0;
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) own += w[e] = entry(n, e) < min(n, most) ? weight_of(key[e]) : 0ull;
        before = above + dc_before(own, sh.wsum, all);
        sum = above + all;
        P = share > 0.f ? dw_share(share, total ? total : sum) : ~0ull;
        int kept = 0;
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) {
            const u64 x = w[e];
            const bool k = x && before < P;
            if (!k) w[e] = 0;
            kept += __syncthreads_count(k);
            before += x;
        }
        return kept;
    }

    // The draw among listed entries alone: an entry is kept where its weight is not 0.
    __device__ __forceinline__ void draw_list(const u64 (&key)[kDcPer], u64 (&w)[kDcPer], int n, int kept) {
        u64 own = 0, total;
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) {
            if (w[e] && !(dw_value((uint32_t)(key[e] >> 32)) >= min_l)) w[e] = 0;
            own += w[e];
        }
        (void)dc_before(own, sh.wsum, total);
        const u64 U = dw_target(A.u[row], total);
        u64* ws = sh.mine;
        if (kept <= 128) {
            // running sums in vocabulary order by comparing indices
#pragma unroll
            for (int e = 0; e < kDcPer; ++e)
                if (entry(n, e) < kept) ws[entry(n, e)] = w[e];
            __syncthreads();
            if (tid < kept) {
                const u64 k = sh.list[tid];
                const uint32_t inv = (uint32_t)k;
                u64 before = 0;
#pragma unroll 4
                for (int j = 0; j < kept; ++j) before += (uint32_t)sh.list[j] > inv ? ws[j] : 0ull;
                if (ws[tid] && before <= U && before + ws[tid] > U) dw_result(A, row, ~inv, dw_logprob(r, dw_value((uint32_t)(k >> 32)), total));
            }
            return;
        }
        // sorted by their index (~index << 32 | place: a rising index is a falling word), then prefix sums
        __syncthreads();
        for (int i = tid; i < kept; i += kDwThreads) ws[i] = (u64)(uint32_t)sh.list[i] << 32 | (uint32_t)i;
        __syncthreads();
        dc_sort(ws, kept);
        u64 v[kDcPer], sum = 0, all;
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) {
            const int i = entry(kept, e);
            const float l = i < kept ? dw_value((uint32_t)(sh.list[(uint32_t)ws[i]] >> 32)) : -INFINITY;
            sum += v[e] = l >= min_l ? weight(l) : 0ull;
        }
        u64 before = dc_before(sum, sh.wsum, all);
#pragma unroll
        for (int e = 0; e < kDcPer; ++e) {
            if (v[e] && before <= U && before + v[e] > U) {
                const u64 k = sh.list[(uint32_t)ws[entry(kept, e)]];
                dw_result(A, row, ~(uint32_t)k, dw_logprob(r, dw_value((uint32_t)(k >> 32)), total));
            }
            before += v[e];
        }
    }

    // (On the first CTA.)  The first m of the logits that are v, of which the warps' stretches have sh.ties: their weights to sh.segs, and the last one's key.
    __device__ __forceinline__ u64 cut_of_ties(float v, u64 m, u64 w) {
        if (warp == 0) {
            const int n = S * kDwWarps;
            const int n0 = 2 * lane < n ? sh.ties[2 * lane] : 0, n1 = 2 * lane + 1 < n ? sh.ties[2 * lane + 1] : 0;
            int upto = n0 + n1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            const int from = upto - n0 - n1, k0 = min(n0, max(0, (int)m - from)), k1 = min(n1, max(0, (int)m - from - n0));
            if (k0) sh.segs[2 * lane] += (u64)k0 * w;
            if (k1) sh.segs[2 * lane + 1] += (u64)k1 * w;
            if (from < (int)m && upto >= (int)m) {
                sh.found = 2 * lane + (k1 > 0);
                sh.n_in = k1 > 0 ? k1 : k0;
            }
        }
        __syncthreads();
        const int f = sh.found, need = sh.n_in, c = f / kDwWarps;
        const T* lg = reinterpret_cast<const T*>(A.logits) + (size_t)row * A.ld;
        const int lo = f % kDwWarps * seg + (int)((unsigned)seg * (unsigned)tid / (unsigned)kDwThreads),
                  hi = f % kDwWarps * seg + (int)((unsigned)seg * (unsigned)(tid + 1) / (unsigned)kDwThreads);
        u64 own = 0, all;
        uint32_t index = 0;
#pragma unroll 1
        for (int turn = 0; turn < 2; ++turn) {
            int at_most = turn ? need - (int)own : 0x7FFFFFFF;
            u64 seen = 0;
#pragma unroll 1
            for (int i = lo; i < hi && (int)seen < at_most; ++i) {
                const int at = c * n_slice + i - off;
                if (at >= 0 && at < A.V && dw_f32(lg[at]) == v) ++seen, index = (uint32_t)at;
            }
            if (!turn) {
                own = dc_before(seen, sh.wsum, all);
                if (!((int)own < need && (int)(own + seen) >= need)) break;
            } else {
                sh.first = index;
            }
        }
        __syncthreads();
        return (u64)dw_key(v) << 32 | (uint32_t)~sh.first;
    }

    // The draw among all logits down to `cut` (key << 32 | ~index) and min_l, from the weights of the warps' stretches in sh.segs, to which those of the first
    // `kept` listed entries are added.  `alone`: one CTA for the row, with that stretch from global memory; otherwise the CTA that has it.  False: they are over
    // `limit`.
    __device__ __forceinline__ bool draw_segments(u64 cut, int kept, bool alone, u64 limit) {
        const int n = S * kDwWarps;
#pragma unroll 1
        for (int i = tid; i < kept; i += kDwThreads) {
            const u64 k = sh.list[i];
            const int place = (int)~(uint32_t)k + off;
            if (dw_value((uint32_t)(k >> 32)) >= min_l) atomicAdd(&sh.segs[place / n_slice * kDwWarps + place % n_slice / seg], weight_of(k));
        }
        __syncthreads();
        if (warp == 0) {  // (up to two stretches a lane)
            const u64 w0 = 2 * lane < n ? sh.segs[2 * lane] : 0ull, w1 = 2 * lane + 1 < n ? sh.segs[2 * lane + 1] : 0ull;
            u64 upto = w0 + w1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            const u64 all = __shfl_sync(0xffffffffu, upto, 31), from = upto - w0 - w1;
            if (all <= limit) {
                const u64 U = dw_target(A.u[row], all);
                if (from <= U && upto > U) {
                    const bool second = from + w0 <= U;
                    sh.found = 2 * lane + second;
                    sh.before = second ? from + w0 : from;
                    sh.target = U;
                }
            }
            if (lane == 0) sh.sum = all;
        }
        __syncthreads();
        const u64 total = sh.sum;
        if (total > limit) return false;
        const u64 U = sh.target;
        const int f = sh.found, c = f / kDwWarps;
        if (c != rank && !alone) return true;
        // that stretch again: consecutive logits per thread
        const T* lg = reinterpret_cast<const T*>(A.logits) + (size_t)row * A.ld;
        const int lo = f % kDwWarps * seg + (int)((unsigned)seg * (unsigned)tid / (unsigned)kDwThreads),
                  hi = f % kDwWarps * seg + (int)((unsigned)seg * (unsigned)(tid + 1) / (unsigned)kDwThreads);
        u64 b = 0;
#pragma unroll 1
        for (int turn = 0; turn < 2; ++turn) {
            u64 sum = 0;
#pragma unroll 1
            for (int i = lo; i < hi; ++i) {
                const int at = c * n_slice + i - off;
                const float l = c == rank ? dw_f32(slice[i]) : at >= 0 && at < A.V ? dw_f32(lg[at]) : -INFINITY;
                if (!(l >= min_l && ((u64)dw_key(l) << 32 | (uint32_t)~(uint32_t)at) >= cut)) continue;
                const u64 x = weight(l);
                sum += x;
                if (turn) {
                    b += x;
                    if (b > U) {
                        dw_result(A, row, (uint32_t)at, dw_logprob(r, l, total));
                        break;
                    }
                }
            }
            if (turn) return true;
            u64 all;
            b = sh.before + dc_before(sum, sh.wsum, all);
            if (!(sum && b <= U && b + sum > U)) return true;
        }
        return true;
    }

    __device__ __forceinline__ void finish(DcEnd end, DcCut c) {
        if (end == kDcByMinP) {
            double own = 0;
            scan([&](const float (&v)[N], float largest, int, int) {
                weights(v, largest, min_l, [&](float l, double w) {
                    if (l >= min_l) own += w;
                });
            });
            const u64 sum = dc_warp_sum((u64)own);
            if (lane < S) dc_put(lane, &sh.segs[rank * kDwWarps + warp], sum);
            dc_sync(S);
            c.cut = 0, c.kept = 0;
        }
        if (end == kDcByMinP || end == kDcByCut)
            if (!draw_segments(c.cut, c.kept, end == kDcByCut, c.limit)) end = kDcByPasses;
        if (end == kDcByPasses && rank == 0) dw_row_plain<T>(A, row, *reinterpret_cast<DwPlainShared*>(slice));
    }
};

// A stretch of values that a cut lies in, and its histogram.
template <typename T>
struct DcStretch {
    DcRow<T>& R;
    static constexpr int N = DcVec<T>::n;
    float mn;               // the smallest of the threads' largest logits
    bool marked, weighed;   // marked: the slice is short enough for marks; weighed: the bins are (for top-p)
    float rel_unit;         // (8192 or, of 16 bits, 16384 logits of a marked slice stay under 2^32, and up to 98304 of a long one)
    float from_l, to_l;     // the cut lies from here on, under this
    const u64* base;        // weights of the warps' stretches from to_l on (null: none),
    u64 base_all, base_n;   // of all, and their number (for top-k's cut)
    uint32_t marks[N / 4];  // logits from from_l on
    float top_l, per_bin, bin_y;  // (bin_y: what y changes by from bin to bin)
    uint32_t cnt[kDcBinsPer];
    u64 rel[kDcBinsPer];

    __device__ __forceinline__ void begin(float smallest) {
        mn = smallest;
        marked = R.seg <= 32 * N * kDcMarked;
        weighed = R.r.top_p > 0.f;
        rel_unit = marked ? 131072.0f : 16384.0f;
    }
    __device__ __forceinline__ void whole(float from) { from_l = from, to_l = INFINITY, base = nullptr, base_all = base_n = 0; }
    __device__ __forceinline__ void mark() {
        if (!marked) return;
#pragma unroll
        for (int g = 0; g < N / 4; ++g) marks[g] = 0;
        R.scan([&](const float (&v)[N], float largest, int, int i) {
            if (largest >= from_l) R.mark(marks, v, i, from_l);
        });
    }
    // The bins of a stretch that ends with logits (`known`), or of one that may reach far down: no further then than 2.5 times the range of the threads' largest logits, unless
    // those are all the same.
    __device__ __forceinline__ void set_bins(bool known) {
        top_l = fminf(to_l, R.r.mx);
        const float most = 2.5f * (R.r.mx - mn), span = fminf(top_l - from_l, !known && most > 0.f ? most : 3.402823466e38f);
        per_bin = span > 0.f ? fminf(((float)kDcBins - 1.0f) / span, 1e30f) : 1e30f;
        bin_y = -(float)R.r.c / per_bin;
    }
    // The bin of a logit from from_l on and under to_l; in the last one: all that is further down.
    __device__ __forceinline__ float where(float l) const { return fminf((top_l - l) * per_bin, (float)kDcBins - 0.5f); }
    __device__ __forceinline__ bool in(float l) const { return l >= from_l && l < to_l; }
    // All CTAs' histograms, two bins a thread.
    __device__ __forceinline__ void count() {
        R.each(marks, [&](const float (&l)[4], const int (&)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (in(l[e])) {
                    const float q = where(l[e]);
                    const int i = (int)q;
                    atomicAdd(&R.sh.hist[i].x, 1u);
                    if (weighed) atomicAdd(&R.sh.hist[i].y, (uint32_t)(exp2f((q - (float)i) * bin_y) * rel_unit));
                }
        });
        dc_sync(R.S);
#pragma unroll
        for (int i = 0; i < kDcBinsPer; ++i) cnt[i] = 0, rel[i] = 0;
#pragma unroll
        for (int c = 0; c < kDcMaxCtas; ++c)
            if (c < R.S) {
                const uint4 h = dc_u32x4(&R.sh.hist[kDcBinsPer * R.tid], c);
                cnt[0] += h.x, cnt[1] += h.z;
                rel[0] += h.y, rel[1] += h.w;
            }
    }
    // The bins where the running sum reaches `want` and `to`, b1 and b2, and the number of logits from the one to the other.
    template <typename V>
    __device__ __forceinline__ int find_bins(u64 before, const V (&v)[kDcBinsPer], u64 want, u64 to, int& b1, int& b2) {
        DcShared& sh = R.sh;
        if (R.tid == 0) sh.bin = sh.bin_to = kDcBins - 1, sh.n_in = 0;
        __syncthreads();
        u64 at = before;
        if (R.tid == 0 && before >= want) sh.bin = 0;
#pragma unroll
        for (int i = 0; i < kDcBinsPer; ++i) {
            const u64 next = at + (u64)v[i];
            if (at < want && next >= want) sh.bin = kDcBinsPer * R.tid + i;
            if (at < to && next >= to) sh.bin_to = kDcBinsPer * R.tid + i;
            at = next;
        }
        __syncthreads();
        b1 = sh.bin, b2 = sh.bin_to;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kDcBinsPer; ++i)
            if (kDcBinsPer * R.tid + i >= b1 && kDcBinsPer * R.tid + i <= b2) n += (int)cnt[i];
        n = __reduce_add_sync(0xffffffffu, n);
        if (R.lane == 0 && n) atomicAdd(&sh.n_in, n);
        __syncthreads();
        return sh.n_in;
    }
    // Top-k's cut: whether there is one here, and its bin (kDcBins: none).
    __device__ __forceinline__ bool find_k(int& b1, int& n_in) {
        u64 sum = 0, all;
#pragma unroll
        for (int i = 0; i < kDcBinsPer; ++i) sum += cnt[i];
        const u64 before = base_n + dc_before(sum, R.sh.wsum, all);
        b1 = kDcBins, n_in = 0;
        if (base_n + all < (u64)R.r.top_k) return false;
        int b2;
        n_in = find_bins(before, cnt, R.r.top_k, R.r.top_k, b1, b2);
        return true;
    }
    // Top-p's cut: between the bins that the bins' weights say, in units of 2^-24 of the largest one here.
    __device__ __forceinline__ int find_p(u64 P, int& b1, int& b2) {
        const DwRow& r = R.r;
        const double unit = exp2(24.0 - (double)r.F + (r.mxd - (double)top_l) * r.c);
        const float scale = 16777216.0f / rel_unit;
        float near[kDcBinsPer];
        u64 sum = 0, all;
#pragma unroll
        for (int i = 0; i < kDcBinsPer; ++i) {
            near[i] = rintf((float)rel[i] * exp2f((float)(kDcBinsPer * R.tid + i) * bin_y) * scale);
            sum += (u64)near[i];
        }
        const u64 before = dc_before(sum, R.sh.wsum, all), want = P > base_all ? (u64)fmin((double)(P - base_all) * unit, 1e18) : 0ull;
        // A logit's weight in its bin is cut at 2^-17 (or 2^-14) of the bin's upper end.  (Bins that are only counted, with the weight of their middle, made
        // rows of 1024 x 65536 with top-p 0.9 1 % faster, but missed the cut where logits have few values: one bf16 row in some hundreds, of 1 ms.)
        const u64 off = (want >> (marked ? 15 : 12)) + 512;
        return find_bins(before, near, want > off ? want - off : 1, want + off, b1, b2);
    }
    // min-p's cut comes before bin b.
    __device__ __forceinline__ bool min_p_before(int b) const { return where(R.min_l) < (float)b || R.min_l >= to_l; }

    // The weights of the warps' stretches in front of bins b1 .. b2 to segs, their number to above, and the logits of the bins to list number c, all in the first
    // CTA; or (ZOOM) what they weigh and how many they are together, and the largest and the smallest in the bins, to all CTAs.
    template <bool ZOOM>
    __device__ __forceinline__ void region(int c, int b1, int b2) {
        DcShared& sh = R.sh;
        const int rank = R.rank, warp = R.warp, lane = R.lane;
        const float q1 = (float)b1, q2 = (float)(b2 + 1);
        double own = 0;
        int above = 0, n = 0;
        float hi = -INFINITY, lo = INFINITY;
        R.each(marks, [&](const float (&l)[4], const int (&at)[4]) {
            double w[4];
            bool a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = in(l[e]) && where(l[e]) < q1;
            if (__any_sync(0xffffffffu, a[0] || a[1] || a[2] || a[3])) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = dw_whole(R.r, l[e], sh.tab);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (a[e]) own += w[e], ++above;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!a[e] && in(l[e]) && where(l[e]) < q2) {
                    if (ZOOM)
                        hi = fmaxf(hi, l[e]), lo = fminf(lo, l[e]), ++n;
                    else
                        R.collect(l[e], at[e]);
                }
        });
        const u64 sum = dc_warp_sum((u64)own) + (base ? base[warp] : 0ull);
        above = __reduce_add_sync(0xffffffffu, above);
        if (lane == 0) {
            dc_put(0, &sh.segs[rank * kDwWarps + warp], sum);
            sh.n_above[warp] = above;
        }
        if (ZOOM) {
            n = __reduce_add_sync(0xffffffffu, n);
            hi = dc_warp_max(hi), lo = dc_warp_min(lo);
            if (lane == 0) {
                dc_put(0, &sh.ties[rank * kDwWarps + warp], n);
                sh.seg_a[warp] = sum;
                sh.red[warp] = hi, sh.redmin[warp] = lo;
            }
            __syncthreads();
            if (warp == 0) {
                const u64 t = dc_all(sh.seg_a[lane & 7], DcAdd());
                const int all = dc_all(sh.n_above[lane & 7], DcAdd());
                hi = dc_warp_max(sh.red[lane & 7]), lo = dc_warp_min(sh.redmin[lane & 7]);
                if (lane < R.S) {
                    dc_put(lane, &sh.sums[rank].total, t);
                    dc_put(lane, &sh.sums[rank].n, (u64)all);
                    dc_put(lane, &sh.top[rank], make_float4(hi, lo, 0.f, 0.f));
                }
            }
        } else {
            R.hand_in(c);
            if (R.tid == 0) {
                int t = 0;
#pragma unroll
                for (int i = 0; i < kDwWarps; ++i) t += sh.n_above[i];
                dc_put(0, &sh.above[rank], t);
            }
        }
        dc_sync(R.S);
    }
    // (All CTAs.)  Top-k's cut in bin b1 (!here: further down than all logits here), with top-p's where that comes later.  False: top-p's lies further up, before P.
    __device__ __forceinline__ bool cut_at_k(int b1, bool here, u64& total, u64& P, DcEnd& end, DcCut& c) {
        DcShared& sh = R.sh;
        const DwRow& r = R.r;
        region<false>(1, b1, b1);
        end = kDcDone;
        if (R.rank != 0) {
            if (r.top_p <= 0.f) return true;
            dc_sync(R.S);
        } else {
            u64 key[kDcPer], w[kDcPer], above = 0;
            const int n = sh.n_list[1];
            (void)dc_before(R.tid < R.S * kDwWarps ? sh.segs[R.tid] : 0ull, sh.wsum, above);
            const int n_above = (int)base_n + dc_all((R.lane & 7) < R.S ? sh.above[R.lane & 7] : 0, DcAdd());
            const bool fits = n <= kDcList;
            if (fits) {
                R.sorted(n, key);
                c.kept = R.cut_of(key, n, here ? (int)r.top_k - n_above : 0, above, r.top_p, 0, w, P, total);
                c.cut = c.kept ? sh.list[c.kept - 1] : 0ull;
            }
            end = fits ? kDcByCut : kDcByPasses;
            if (r.top_p <= 0.f) return true;  // (the others have left)
            // Where top-p's cut lies further up the others are told what it is a share of.
            const bool done = !fits || above < P;
            const bool by_min = fits && above < P && min_p_before(b1);  // top-p's cut is here, min-p's further up
            if (R.tid < R.S) {
                dc_put(R.tid, &sh.left, total);
                dc_put(R.tid, &sh.cut_p, by_min ? ~0ull : done ? 0ull : P);
            }
            dc_sync(R.S);
        }
        total = sh.left;
        P = sh.cut_p;
        if (P == ~0ull) end = kDcByMinP;
        return P == 0 || P == ~0ull;
    }
    // Top-p's cut in bins b1 .. b2.
    __device__ __forceinline__ DcEnd cut_at_p(int b1, int b2, u64 total, u64 P, DcCut& c) {
        DcShared& sh = R.sh;
        region<false>(2, b1, b2);
        if (R.rank != 0) return kDcDone;
        const int n = sh.n_list[2];
        u64 above = 0;
        (void)dc_before(R.tid < R.S * kDwWarps ? sh.segs[R.tid] : 0ull, sh.wsum, above);
        if (n > kDcList || above >= P) return kDcByPasses;
        u64 key[kDcPer], w[kDcPer], P2, upto;
        R.sorted(n, key);
        c.kept = R.cut_of(key, n, n, above, R.r.top_p, total, w, P2, upto);
        if (upto < P) return kDcByPasses;  // the cut lies further down
        c.cut = sh.list[c.kept - 1];
        return kDcByCut;
    }
};

// A cut whose bins b1 .. b2 of the stretch from_l .. to_l hold n_in logits, too many to sort: they are divided into 512 bins again, and so on.  (All CTAs of the
// row.  A function of its own, which begins with what is in shared memory, so that the rows without it have its registers.)
template <typename T>
__device__ __noinline__ void dc_zoomed(const DrawArgs& A, int S, int n_slice, bool by_k) {
    extern __shared__ __align__(16) unsigned char dc_smem[];
    DcShared& sh = *reinterpret_cast<DcShared*>(dc_smem);
    DcRow<T> R = {A, sh, reinterpret_cast<T*>(dc_smem + sizeof(DcShared))};
    R.tid = threadIdx.x, R.lane = R.tid & 31, R.warp = R.tid >> 5;
    R.S = S;
    R.rank = S > 1 ? (int)dc_rank() : 0;
    R.row = (int)blockIdx.x / S;
    R.n_slice = n_slice;
    R.seg = n_slice / kDwWarps;
    R.off = (int)((reinterpret_cast<uintptr_t>(reinterpret_cast<const T*>(A.logits) + (size_t)R.row * A.ld) & 15) / sizeof(T));
    R.r = dw_asked(A, R.row);
    DwRow& r = R.r;
    __syncthreads();
    r.mx = sh.zoom.mx, r.mxd = (double)r.mx, r.c = sh.rate, r.ymin = sh.least;
    R.floor_l = sh.floor_l, R.min_l = sh.min_l;
    DcStretch<T> D = {R};
    D.begin(sh.zoom.mn);
    const float from_all = sh.zoom.from_l;
    D.whole(from_all);
    D.to_l = sh.zoom.to_l, D.base = sh.zoom.base, D.base_all = sh.zoom.base_all;
    D.mark();
    D.set_bins(false);  // (as they were)
    u64 total = sh.zoom.total;
    int b1 = sh.bin, b2 = sh.bin_to, n_in = sh.n_in;
    __syncthreads();
    u64 P = by_k ? 0ull : dw_share(r.top_p, total);
    int zooms = 0;
    bool here = true;
    DcCut c = {0, ~0ull, 0};
    DcEnd end = kDcByPasses;
#pragma unroll 1
    while (true) {
        bool known = false;
        if (n_in > kDcList) {
            if (zooms++ == kDcZooms) {
                dc_sync(S);  // (the histograms are being read)
                break;
            }
            D.template region<true>(0, b1, b2);
            const bool one = (R.lane & 7) < S;
            D.base = sh.seg_a;
            D.base_all = dc_all(one ? sh.sums[R.lane & 7].total : 0ull, DcAdd());
            D.base_n += dc_all(one ? sh.sums[R.lane & 7].n : 0ull, DcAdd());
            const float hi = dc_warp_max(one ? sh.top[R.lane & 7].x : -INFINITY), lo = dc_warp_min(one ? sh.top[R.lane & 7].y : INFINITY);
            D.from_l = lo, D.to_l = nextafterf(hi, INFINITY);
            known = true;
            if (!(lo < hi)) {
                // equal ones: as many of them as the weight or the number left needs
                const u64 w = R.weight(lo);
                u64 m = by_k ? (u64)r.top_k - D.base_n : (u64)n_in;
                if (by_k && r.top_p > 0.f) total = D.base_all + m * w, P = dw_share(r.top_p, total);
                if (r.top_p > 0.f && D.base_all >= P) {  // top-p's cut lies further up
                    if (!by_k) break;
                    by_k = known = false;
                    D.whole(from_all);
                } else {
                    if (r.top_p > 0.f) {
                        const u64 t = (P - D.base_all + w - 1) / w;
                        if (t > (u64)n_in) break;
                        if (t < m) m = t;
                    }
                    end = R.min_l > lo ? kDcByMinP : R.rank == 0 ? kDcByCut : kDcDone;
                    if (end == kDcByCut) c.cut = R.cut_of_ties(lo, m, w);
                    break;
                }
            }
        } else if (by_k) {
            if (D.cut_at_k(b1, here, total, P, end, c)) break;
            by_k = false;
            end = kDcByPasses, c.kept = 0;
            D.whole(from_all);
        } else {
            end = D.cut_at_p(b1, b2, total, P, c);
            break;
        }
        D.set_bins(known);
        reinterpret_cast<uint4*>(sh.hist)[R.tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        D.count();
        if (by_k) {
            here = D.find_k(b1, n_in);
            b2 = b1;
            if (!here) {
                dc_sync(S);
                break;
            }
            if (!(r.top_p > 0.f) && D.min_p_before(b1)) {
                end = kDcByMinP;
                break;
            }
        } else {
            n_in = D.find_p(P, b1, b2);
            if (D.min_p_before(b1)) {
                end = kDcByMinP, c.limit = P;
                break;
            }
        }
    }
    R.finish(end, c);
}

template <typename T>
__global__ void __launch_bounds__(kDwThreads, 5) draw_cluster_kernel(const __grid_constant__ DrawArgs A, int S, int n_slice) {
    extern __shared__ __align__(16) unsigned char dc_smem[];
    DcShared& sh = *reinterpret_cast<DcShared*>(dc_smem);
    DcRow<T> R = {A, sh, reinterpret_cast<T*>(dc_smem + sizeof(DcShared))};
    constexpr int N = DcVec<T>::n;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = S > 1 ? (int)dc_rank() : 0;
    R.tid = tid, R.lane = lane, R.warp = warp;
    R.S = S;
    R.rank = rank;
    R.row = (int)blockIdx.x / S;
    R.n_slice = n_slice;
    R.seg = n_slice / kDwWarps;
    dc_arrive(S);
    R.r = dw_asked(A, R.row);
    DwRow& r = R.r;

    // ---- the row, its largest logit, bounds of what is kept
    const float tm = R.load([&] {
        uint4* h = reinterpret_cast<uint4*>(sh.hist);
        for (int i = tid; i < kDcBins / 2; i += kDwThreads) h[i] = make_uint4(0, 0, 0, 0);
        sh.tmhist[tid] = 0u;
        dw_fill_table(sh.tab, A.F);
        if (tid == 0) {
            sh.n_list[0] = sh.n_list[1] = sh.n_list[2] = sh.n_mine = 0;
            sh.first = ~0u;
            sh.thr_all = sh.thr_part = -INFINITY;
        }
        if (warp == kDwWarps - 1 && !r.greedy) {
            const double c = dw_rate(r.T), y = dw_least(r.min_p);
            if (lane == 0) sh.rate = c, sh.least = y;
        }
    });
    float mx = dc_warp_max(tm), mn = dc_warp_min(tm > -INFINITY ? tm : INFINITY);
    if (lane == 0) sh.red[warp] = mx, sh.redmin[warp] = mn;
    __syncthreads();
    const bool small = A.V <= kDcList;
    const bool list_k = !r.greedy && !small && r.top_k && r.top_k <= (uint32_t)min(kDcFastK, S * kDcMostPart);
    const bool list_p = !r.greedy && !small && !r.top_k && r.top_p > 0.f;
    const bool list = !r.greedy && (small || list_k || list_p);
    const bool binned_k = !r.greedy && !list && r.top_k;
    mx = dc_warp_max(sh.red[lane & (kDwWarps - 1)]);
    mn = dc_warp_min(sh.redmin[lane & (kDwWarps - 1)]);
    if (list_k || list_p || binned_k) R.bounds(tm, mx, mn, list_p ? min(kDcTryK, S * kDcTryPart) : (int)r.top_k);
    dc_wait(S);
    if (tid < S) dc_put(tid, &sh.top[rank], make_float4(mx, mn, sh.thr_all, sh.thr_part));
    dc_sync(S);
    float thr;
    int owner;  // the first CTA with the largest logit
    {
        const float4 t = (lane & 7) < S ? sh.top[lane & 7] : make_float4(-INFINITY, INFINITY, -INFINITY, INFINITY);
        mx = dc_warp_max(t.x);
        mn = dc_warp_min(t.y);
        thr = fmaxf(fmaxf(dc_warp_max(t.z), dc_warp_min(t.w)), -3.402823466e38f);  // (-inf is never drawn)
        owner = __ffs(__ballot_sync(0xffffffffu, t.x == mx)) - 1;
    }
    if (!(mx > -INFINITY)) {  // (a NaN, or nothing to draw)
        if (rank == 0 && tid == 0) dw_result(A, R.row, kDwNone, mx);
        return;
    }
    if (r.greedy) {
        if (rank != owner) return;
        uint32_t best = kDwNone;
        R.scan([&](const float (&v)[N], float, int place, int) {
#pragma unroll
            for (int e = N - 1; e >= 0; --e)
                if (v[e] == mx) best = min(best, (uint32_t)(place + e));
        });
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0) atomicMin(&sh.first, best);
        __syncthreads();
        if (tid == 0) dw_result(A, R.row, R.index_of((int)sh.first), 0.f);
        return;
    }
    if (mx == INFINITY) return R.finish(kDcByPasses, {});
    r.mx = mx;
    r.mxd = (double)mx;
    r.c = sh.rate;
    r.ymin = sh.least;
    if (warp == 0) {
        const float a = dc_threshold(r, -40.0), b = r.ymin > -40.0 ? dc_threshold(r, r.ymin) : a;
        if (lane == 0) sh.floor_l = a, sh.min_l = b;
    }
    __syncthreads();
    R.floor_l = sh.floor_l;
    R.min_l = sh.min_l;

    // ---- list
    bool binned_p = false, done_marks = false;
    u64 total = 0;  // weight of all that top-k leaves
    DcStretch<T> D = {R};
    D.begin(mn);
    D.whole(thr);
#pragma unroll
    for (int g = 0; g < N / 4; ++g) D.marks[g] = 0;
    if (list) {
        // the smallest of the threads' maxima bounds the other stretches of values: a fifth of normally distributed logits is larger
        const float l_a = fmaxf(thr, R.floor_l), l_c = fmaxf(fminf(mn, thr), R.floor_l);
        double own = 0, own_a = 0, own_c = 0;
        R.scan([&](const float (&v)[N], float largest, int place, int i) {
            if (largest >= thr)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (v[e] >= thr) R.collect(v[e], place + e);
            if (list_p) {
                R.weights(v, largest, R.floor_l, [&](float l, double w) {
                    if (l >= R.floor_l) own += w;
                    if (l >= l_a) own_a += w;
                    if (l >= l_c) own_c += w;
                });
                if (D.marked) R.mark(D.marks, v, i, l_c);
            }
        });
        if (list_p) {
            const u64 sum = dc_warp_sum((u64)own), sum_a = dc_warp_sum((u64)own_a), sum_c = dc_warp_sum((u64)own_c);
            if (lane == 0) sh.wsum[warp] = sum, sh.seg_a[warp] = sum_a, sh.seg_c[warp] = sum_c;
            __syncthreads();
            if (warp == 0) {  // (eight lanes add up the warps of one sum each)
                const u64* p = lane < 8 ? sh.wsum : lane < 16 ? sh.seg_a : sh.seg_c;
                const u64 t = dc_all(p[lane & 7], DcAdd());
                u64* to = lane < 8 ? &sh.sums[rank].total : lane < 16 ? &sh.sums[rank].from_a : lane < 24 ? &sh.sums[rank].from_c : &sh.sums[rank].n;
                if ((lane & 7) < S) dc_put(lane & 7, to, lane < 24 ? t : (u64)sh.n_mine);
            }
        }
        R.hand_in(0);
        dc_sync(S);
        if (list_p) {
            const bool one = (lane & 7) < S;
            const DcSums& o = sh.sums[lane & 7];
            total = dc_all(one ? o.total : 0ull, DcAdd());
            const u64 sum_a = dc_all(one ? o.from_a : 0ull, DcAdd()), sum_c = dc_all(one ? o.from_c : 0ull, DcAdd());
            const u64 P = dw_share(r.top_p, total);
            const bool over = dc_all(one ? o.n : 0ull, DcAdd()) > (u64)kDcList;
            binned_p = over || P > sum_a;
            done_marks = P <= sum_c;
            D.from_l = l_c, D.to_l = l_a, D.base = sh.seg_a, D.base_all = sum_a;
            if (P <= sum_a) D.whole(l_c);
            if (P > sum_c) D.from_l = R.floor_l, D.to_l = l_c, D.base = sh.seg_c, D.base_all = sum_c;
        }
        if (!binned_p) {
            if (rank != 0) return;
            const int n = sh.n_list[0];
            if (n > kDcList || n < (int)(list_k ? r.top_k : 0u)) {
                // (fewer than top-k asks for: there are no more, or the bound was rounded up)
                if (n > kDcList || thr > -3.402823466e38f) return R.finish(kDcByPasses, {});
            }
            u64 key[kDcPer], w[kDcPer], P, sum;
            R.sorted(n, key);
            const int kept = R.cut_of(key, n, r.top_k ? (int)r.top_k : n, 0, r.top_p, total, w, P, sum);
            R.draw_list(key, w, n, kept);
            return;
        }
    }
    D.from_l = fmaxf(D.from_l, R.floor_l);

    // ---- region
    DcCut c = {0, ~0ull, 0};
    DcEnd end = kDcByMinP;
    if (binned_p || binned_k) {
        D.set_bins(false);
        if (!done_marks) D.mark();
        D.count();
        int b1, b2, n_in = 0;
        u64 P = 0;
        bool at_p = !binned_k, zoom = false;
        if (binned_k) {
            // Where fewer logits have a weight (or the bound was rounded up) there is no cut of top-k among them.
            const bool here = D.find_k(b1, n_in);
            if (!here && thr >= R.floor_l) {
                dc_sync(S);  // (the histograms are being read)
                end = kDcByPasses;
            } else if (r.top_p > 0.f || !D.min_p_before(b1)) {  // (otherwise min-p's cut is the stricter one)
                zoom = n_in > kDcList;
                if (!zoom) at_p = !D.cut_at_k(b1, here, total, P, end, c);
            }
        } else {
            P = dw_share(r.top_p, total);
        }
        if (at_p) {
            n_in = D.find_p(P, b1, b2);
            end = kDcByMinP;
            if (D.min_p_before(b1)) {
                c.limit = P;
            } else {
                zoom = n_in > kDcList;
                if (!zoom) end = D.cut_at_p(b1, b2, total, P, c);
            }
        }
        if (zoom) {
            if (tid == 0) sh.zoom = {mx, D.mn, D.from_l, D.to_l, D.base, D.base_all, total};
            return dc_zoomed<T>(A, S, n_slice, !at_p);
        }
        if (end == kDcDone) return;
    }
    R.finish(end, c);
}

}  // namespace rsv
