// Low-rank adapters of many requests at once, beside a projection that all rows share:
//   out[n] = base[n] + scale[a] B[a] (A[a] x[n]),  a = index[n]; rows with an index outside 0 .. slots - 1 have no adapter: out[n] = base[n].
//
// One launch, no work area.  A cluster of CTAs takes a tile: up to 16 MT rows of one adapter, wherever they lie.  Which ones follows from the indices
// alone: every cluster counts the rows per adapter, numbers the tiles adapter by adapter and gathers the rows of its own (of 4096 rows at a time, so that
// this stays short).  So an adapter is read once per tile, not once per row, and the host need not know the indices.
//   t = A x   the CTAs of the cluster split K, the warps of a CTA split it again; the partial sums meet in shared memory and then in the cluster's.
//   B t       the CTAs split M; every CTA has all of t.
// Both products run on the tensor cores with fp32 sums.  16-bit activations are operands as they are; fp32 ones are two tf32 numbers each (ad_split),
// and the 16-bit weights are exact in tf32.  t is two fp16 numbers per value, or two bf16 ones (2^-17 of it off; three, 2^-25, where out is fp32), so that B is an
// operand as it is.  fp16 ends early: the row's largest value is brought to 2^14 .. 2^15, and one down to 2^-20 of it is at most 2^-20 of itself off (2^-23 and 2^-17
// where out has 16 bits).  A tile with a value further down whose parts are all that small (one that cancelled is no more exact than its parts), or with a row's largest
// outside 2^-100 .. 2^100, has t as two tf32 numbers (2^-22 of any value) and the second product in tf32: what a rank adds keeps its precision whatever the other
// ranks add, as it has to where outputs use few of them.  (With all tiles of that kind: one fp32 session of 2560 x 2560 11.2 us instead of 8.4, 512 rows with 64 ranks of
// 2560 x 10240 39 instead of 25.)
// The tensor cores line products up by the exponents of their operands, which is that of 2^-14 for all fp16 numbers below: the sums of B t (and of A x, where x is fp16) are as exact
// as with weights of 2^-14 where those are smaller (two ranks 2^12 apart with weights of 2^-24 and 3e-5: 2^-14 of their sum off; zeros do not count, and tf32 has no such end).
//
// Bound by its instructions: a scheduler issues in 34 to 53 % of the cycles, four warps of it waiting for fixed latencies, and in short calls for instructions that
// are fetched for the first time.  4096 bf16 rows, 16 adapters of 64 ranks, 2560 x 10240: 75 us, 2.7 TB/s (the second product 50 of them); 64 sessions of 10240 k with 64
// adapters of 16 ranks, fp32: 20 us, 1.0 TB/s; one session of 2560 x 2560: 10 us, all latency.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace rsv {

struct AdapterArgs {
    const void* x;
    const int32_t* index;
    const void *a, *b;  // [slots][max_rank][K], [slots][M][max_rank]
    const int32_t* ranks;  // may be null: max_rank
    const float* scales;   // may be null: 1
    const void* base;      // may be null: 0
    void* out;
    int64_t ldx, ldbase, ldout, a_slot, a_row, b_slot, b_row;
    int rows, K, M, slots, max_rank;
    // launch
    int S, tiles, block_rows, rank_cap;  // CTAs of a cluster; tiles and rows of a block of rows; max_rank rounded up to 16
    int wide_x, wide_a, wide_b, wide_base;  // rows start at 16 bytes
    int wide_out;                           // four values at a time may be stored
    int copies;                            // rows without adapter are written
};

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdMaxRows = 1 << 25;  // (8192 blocks of rows with up to 4096 tiles each, as many CTAs)
constexpr int kAdBlockRows = 4096;
constexpr int kAdMaxCtas = 8;
constexpr int kAdChunk = 64;  // ranks whose sums a warp holds at a time

constexpr size_t kAdSumBytes = (size_t)kAdWarps * 16 * (kAdChunk + 8) * 4;
constexpr int kAdMostCells = 8192;  // rows x rank_cap of a tile: t lies where the sums were
constexpr int kAdGroupAt = kAdMaxSlots + 64;  // the groups of the rows behind the counters
static_assert((kAdGroupAt + kAdBlockRows) * 2 <= kAdSumBytes && kAdMostCells * 4 <= kAdSumBytes, "the counters lie where the sums go later, and t after them");

__device__ __forceinline__ float ad_f32(float v) { return v; }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename X>
__device__ __forceinline__ X ad_round(float v);
template <>
__device__ __forceinline__ float ad_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half ad_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ad_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ad_lo(uint32_t v, const __half*) { return __half2float(__ushort_as_half((unsigned short)v)); }
__device__ __forceinline__ float ad_hi(uint32_t v, const __half*) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
__device__ __forceinline__ float ad_lo(uint32_t v, const __nv_bfloat16*) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float ad_hi(uint32_t v, const __nv_bfloat16*) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ float4 ad_floats(const float4& v, const float*) { return v; }
template <typename H>
__device__ __forceinline__ float4 ad_floats(const uint2& v, const H* h) { return make_float4(ad_lo(v.x, h), ad_hi(v.x, h), ad_lo(v.y, h), ad_hi(v.y, h)); }
__device__ __forceinline__ uint32_t ad_pack(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t ad_pack(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Four values to p, of which the first n exist; `wide`: all at once, where all exist.
__device__ __forceinline__ void ad_store4(float* p, const float4& v) { *reinterpret_cast<float4*>(p) = v; }
template <typename H>
__device__ __forceinline__ void ad_store4(H* p, const float4& v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(ad_pack(v.x, v.y, p), ad_pack(v.z, v.w, p));
}
template <typename E>
__device__ __noinline__ void ad_store_some(E* p, float4 v, int n) {
    if (n > 0) p[0] = ad_round<E>(v.x);
    if (n > 1) p[1] = ad_round<E>(v.y);
    if (n > 2) p[2] = ad_round<E>(v.z);
    if (n > 3) p[3] = ad_round<E>(v.w);
}
template <typename E>
__device__ __forceinline__ void ad_store4(E* p, const float4& v, int n, bool wide) {
    if (wide && n >= 4)
        ad_store4(p, v);
    else
        ad_store_some(p, v, n);
}

// Four 8 x 8 matrices of 16-bit values, a row's address from every lane: an operand of 16 x 16, or two of 8 x 16.
__device__ __forceinline__ void ad_ldm(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
// v as two tf32 numbers: the first rounded to nearest, the rest (of up to 12 bits) cut to 11, so together they are at most 2^-22 of v off and 2^-24 on average.
// The first is always finite: next to the largest float it is the largest tf32 number, and infinities and NaN are in the rest.  (The conversion instruction takes several
// times as long as this.)
__device__ __forceinline__ void ad_split(float v, uint32_t& hi, uint32_t& lo) {
    const float most = __uint_as_float(0x7F7FE000u), h = fminf(fmaxf(__uint_as_float((__float_as_uint(v) + 0x1000u) & 0xFFFFE000u), -most), most);
    hi = __float_as_uint(h);
    lo = __float_as_uint(v - h) & 0xFFFFE000u;
}
__device__ __forceinline__ void ad_mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ad_mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const __half*) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ad_mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const __nv_bfloat16*) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// How a tile of 16 MT rows is worked on: the warps are MT groups of rows times KS parts of K or M.
template <typename X, typename W, int MT, int STAGES>
struct AdShape {
    static constexpr bool wide = sizeof(X) == 4;                                                    // fp32 activations
    static constexpr int pieces = sizeof(X) == 4 && std::is_same<W, __nv_bfloat16>::value ? 3 : 2;  // 16-bit numbers for a value of t
    static constexpr int T = 16 * MT, KS = kAdWarps / MT;
    static constexpr int KC = MT == 1 ? 128 : 64;       // k of a stage
    static constexpr int FW = MT == 4 ? 32 : 16;        // outputs of a warp in a stage
    static constexpr int FB = FW * KS;                  // ... and of a stage
    static constexpr int stages = STAGES;
    static constexpr int most_rank = MT == 1 && STAGES > 3 ? 32 : MT == 4 ? kAdChunk : kAdMaxRank;
    static_assert(T * most_rank <= kAdMostCells, "t lies where the sums were");
    // Bytes from row to row.  16-bit operands are read as matrices of eight rows of 16 bytes: rows an odd multiple of 16 bytes apart lie in different banks.
    // Of the others a lane reads four values of the row that is its number over four: the rows of a quarter (16-byte reads) or half (8-byte reads) of a warp
    // lie in different banks when they are 16 or 8 words apart, modulo 32.
    static constexpr int xld = wide ? (KC + 16) * 4 : (KC + 8) * 2, ald = wide ? (KC + 16) * 2 : (KC + 8) * 2, bld = (FB + 16) * (int)sizeof(X);
    __host__ __device__ static constexpr int stage1(int ranks16) { return T * xld + ranks16 * ald; }
    __host__ __device__ static constexpr int wld(int ranks16) { return (ranks16 + 8) * 2; }
    __host__ __device__ static constexpr int stage2(int ranks16) { return FB * wld(ranks16) + T * bld; }
    __host__ __device__ static constexpr size_t part_bytes(int cap) { return (size_t)T * cap * 4; }
    __host__ __device__ static constexpr size_t piece_bytes(int cap) { return (size_t)pieces * T * wld(cap); }
    __host__ __device__ static constexpr size_t smem(int cap) {
        const int rc = cap < kAdChunk ? cap : kAdChunk, s1 = stage1(rc), s2 = stage2(rc), st = stages * (s1 > s2 ? s1 : s2);
        return 1024 + part_bytes(cap) + piece_bytes(cap) + (st > (int)kAdSumBytes ? st : kAdSumBytes);
    }
};
constexpr int kAdSumLd = kAdChunk + 8;  // (rows eight banks apart)
struct AdTile {
    int rows[64];
    float scale[64];  // 2^e of the row's t, times the adapter's scale
    int slot, n, skip, apart, wsum[kAdWarps];
};
static_assert(sizeof(AdTile) <= 1024, "the tile's part of shared memory");

__device__ __forceinline__ uint32_t ad_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// Sum over the CTA of the values before this thread's (all: the total).
__device__ __forceinline__ int ad_before(int v, int* wsum, int& all) {
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if ((int)(threadIdx.x & 31) >= o) incl += t;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) wsum[threadIdx.x >> 5] = incl;
    __syncthreads();
    int base = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < kAdWarps; ++i) {
        if (i < (int)(threadIdx.x >> 5)) base += wsum[i];
        all += wsum[i];
    }
    return base + incl - v;
}

// The rows of tile `tile` of the block of rows; false: there are fewer tiles.
template <int T>
__device__ __forceinline__ bool ad_find_tile(const AdapterArgs& P, int first, int rows, int tile, AdTile& sh, unsigned short* cnt) {
    const int tid = threadIdx.x, lane = tid & 31, groups = P.slots + 1;  // the last one: rows without adapter
    const int32_t* ix = P.index + first;
    if (rows <= 32) {
        // every warp by itself: a lane has a row, a group is known by its first lane
        const int a = lane < rows ? ix[lane] : -1;
        const int mine = lane >= rows ? P.slots + 1 : a >= 0 && a < P.slots ? a : P.slots;
        const uint32_t same = __match_any_sync(0xffffffffu, mine);
        const bool leads = __ffs(same) - 1 == lane && lane < rows && (mine < P.slots || P.copies);
        const int tiles = leads ? (__popc(same) + T - 1) / T : 0;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, tile >= upto - tiles && tile < upto);
        if (!here) return false;
        const int lead = __ffs(here) - 1, skip = (tile - __shfl_sync(0xffffffffu, upto - tiles, lead)) * T;
        const uint32_t members = __shfl_sync(0xffffffffu, same, lead);
        const int place = __popc(members & ((1u << lane) - 1u)) - skip;
        if (tid < 32) {
            if (members >> lane & 1u && place >= 0 && place < T) sh.rows[place] = first + lane;
            if (lane == lead) sh.slot = mine;
            if (lane == 0) sh.n = min(T, __popc(members) - skip);
        }
        __syncthreads();
        return true;
    }
    unsigned short* group = cnt + kAdGroupAt;  // of every row
    for (int i = tid; i < (groups + 1) / 2; i += kAdThreads) reinterpret_cast<uint32_t*>(cnt)[i] = 0;
    if (tid == 0) sh.slot = -1;
    __syncthreads();
    // (Loops of a few rows rather than all sixteen of a thread unrolled: this runs once, and its instructions have to be fetched.)
#pragma unroll 1
    for (int o = tid; o < rows; o += 4 * kAdThreads) {
        int a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = o + e * kAdThreads < rows ? ix[o + e * kAdThreads] : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (o + e * kAdThreads < rows) {
                const int to = a[e] >= 0 && a[e] < P.slots ? a[e] : P.slots;
                group[o + e * kAdThreads] = (unsigned short)to;
                atomicAdd(reinterpret_cast<uint32_t*>(cnt) + (to >> 1), to & 1 ? 65536u : 1u);  // (no counter passes 4096)
            }
    }
    __syncthreads();
    const int per = (groups + kAdThreads - 1) / kAdThreads, g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    const auto tiles_of = [&](int g) { return g == P.slots && !P.copies ? 0 : ((int)cnt[g] + T - 1) / T; };
    int sum = 0, all;
    for (int g = g0; g < g1; ++g) sum += tiles_of(g);
    int at = ad_before(sum, sh.wsum, all);
    if (tile >= all) return false;
    if (tile >= at && tile < at + sum)
        for (int g = g0; g < g1; ++g) {
            const int t = tiles_of(g);
            if (tile < at + t) {
                sh.slot = g;
                sh.skip = (tile - at) * T;
                sh.n = min(T, (int)cnt[g] - (tile - at) * T);
                break;
            }
            at += t;
        }
    __syncthreads();
    const int mine = sh.slot;
    int n = 0;
#pragma unroll 4
    for (int o = tid; o < rows; o += kAdThreads) n += group[o] == mine;
    int place = ad_before(n, sh.wsum, all) - sh.skip;
    if (n && place < T && place + n > 0)
#pragma unroll 4
        for (int o = tid; o < rows; o += kAdThreads)
            if (group[o] == mine) {
                if (place >= 0 && place < T) sh.rows[place] = first + o;
                ++place;
            }
    __syncthreads();
    return true;
}

// 16 bytes to shared memory, of which the first `bytes` exist (the others are 0).
__device__ __forceinline__ void ad_copy16(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ad_copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void ad_copy(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
// `n` values (none for n <= 0) of a row from src on to 16 bytes of shared memory, zeros behind them; `wide`: src is at 16 bytes.  Rows that are not go in pieces
// of 8 or 4 bytes, asynchronously as well; 16-bit ones that begin inside a word are put together from the words in between.  (4040 rows of 3126 fp32: 117 us value
// by value, 42 so; 1631 rows of 13847 fp32 outputs with 2 ranks: 326 and 152 us.)
template <typename E>
__device__ __noinline__ void ad_fill16(void* dst, const E* src, int n, bool wide) {
    constexpr int N = 16 / (int)sizeof(E);
    if (n <= 0) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
        return;
    }
    const int bytes = min(n, N) * (int)sizeof(E);
    if (wide) {
        ad_copy16(dst, src, bytes);
        return;
    }
    const char* from = reinterpret_cast<const char*>(src);
    const uint32_t at = smem_u32(dst), odd = (uint32_t)reinterpret_cast<uintptr_t>(src);
    if ((odd & 7) == 0) {
        ad_copy<8>(at, from, min(bytes, 8));
        if (bytes > 8)
            ad_copy<8>(at + 8, from + 8, bytes - 8);
        else
            *reinterpret_cast<uint2*>(reinterpret_cast<char*>(dst) + 8) = make_uint2(0, 0);
    } else if ((odd & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            if (bytes > i)
                ad_copy<4>(at + i, from + i, min(bytes - i, 4));
            else
                *reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(dst) + i) = 0;
        }
    } else if constexpr (sizeof(E) == 2) {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(src);
        if (n >= N) {
            const uint32_t first = p[0], w0 = *reinterpret_cast<const uint32_t*>(p + 1), w1 = *reinterpret_cast<const uint32_t*>(p + 3), w2 = *reinterpret_cast<const uint32_t*>(p + 5),
                           last = p[7];
            *reinterpret_cast<uint4*>(dst) = make_uint4(first | w0 << 16, w0 >> 16 | w1 << 16, w1 >> 16 | w2 << 16, w2 >> 16 | last << 16);
        } else {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : 0u;
            *reinterpret_cast<uint4*>(dst) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
        }
    }
}
__device__ __forceinline__ void ad_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ad_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// `count` stages: fill(i, slot) begins to load stage i, use(i, slot) works on it.
template <int STAGES, class Fill, class Use>
__device__ __forceinline__ void ad_pipeline(int count, Fill&& fill, Use&& use) {
#pragma unroll 1  // (the code that begins a stage has to be fetched: twice, not once per stage)
    for (int i = 0; i < STAGES - 1; ++i) {
        if (i < count) fill(i, i);
        ad_commit();
    }
    int slot = 0, next = STAGES - 1;
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
        ad_wait<STAGES - 2>();
        __syncthreads();  // stage i is there for all, and the one before it has been used
        if (i + STAGES - 1 < count) fill(i + STAGES - 1, next);
        ad_commit();
        use(i, slot);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
        next = next + 1 == STAGES ? 0 : next + 1;
    }
    ad_wait<0>();
    __syncthreads();
}

template <typename X, typename W, int MT, int STAGES>
__global__ void __launch_bounds__(kAdThreads, 2) adapters_kernel(AdapterArgs P) {
    typedef AdShape<X, W, MT, STAGES> Z;
    constexpr int T = Z::T, KS = Z::KS, KC = Z::KC, FW = Z::FW, FB = Z::FB, J = FW / 8, pieces = Z::pieces;
    extern __shared__ __align__(16) unsigned char ad_smem[];
    AdTile& sh = *reinterpret_cast<AdTile*>(ad_smem);
    const int cap = P.rank_cap, pld = Z::wld(cap), s1 = Z::stage1(min(cap, kAdChunk));
    float* part = reinterpret_cast<float*>(ad_smem + 1024);
    unsigned char* t16 = ad_smem + 1024 + Z::part_bytes(cap);
    unsigned char* stage = t16 + Z::piece_bytes(cap);
    float* sums = reinterpret_cast<float*>(stage);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3, mt = warp % MT, ks = warp / MT;
    const int S = P.S, rank = S > 1 ? (int)ad_rank() : 0;
    const int job = (int)blockIdx.x / S, block = job / P.tiles, first = block * P.block_rows;
    if (tid == 0) sh.apart = 0;
    if (!ad_find_tile<T>(P, first, min(P.block_rows, P.rows - first), job % P.tiles, sh, reinterpret_cast<unsigned short*>(sums))) return;  // (all CTAs of the cluster)
    const int n_rows = sh.n, a = sh.slot;
    const bool has = a < P.slots;
    const int r_all = !has ? 0 : P.ranks ? max(0, min(__ldg(P.ranks + a), P.max_rank)) : P.max_rank, r16 = (r_all + 15) / 16 * 16;
    const X* xp = reinterpret_cast<const X*>(P.x);
    const X* bp = reinterpret_cast<const X*>(P.base);
    X* op = reinterpret_cast<X*>(P.out);

    float* t32 = reinterpret_cast<float*>(t16);
    static_assert(pieces >= 2, "t fits where its 16-bit numbers go");
    if (r_all > 0) {
        // ---- t = A x: this CTA's part of K, 64 k and more at a time through shared memory
        const int units = (P.K + 63) / 64, k_from = 64 * (int)((long long)units * rank / S), k_to = min(P.K, 64 * (int)((long long)units * (rank + 1) / S));
        const int count = (max(k_to - k_from, 0) + KC - 1) / KC;
        const W* wa = reinterpret_cast<const W*>(P.a) + a * P.a_slot;
#pragma unroll 1
        for (int c0 = 0; c0 < r_all; c0 += kAdChunk) {
            const int ranks = min(kAdChunk, r_all - c0), nt = (ranks + 7) / 8;
            __syncthreads();  // (the counters, or the sums before these, have been read)
            constexpr int XN = 16 / (int)sizeof(X), XU = KC / XN, XP = T * XU / kAdThreads;  // values of 16 bytes, those of a row, and those of a thread
            constexpr int WU = KC / 8, WP = kAdChunk * WU / kAdThreads;
            const int xu = tid % XU * XN, xrow = tid / XU, wu = tid % WU * 8, wrow = tid / WU;
            // (Rows past the tile's last one are not loaded and ranks past the adapter's repeat the last one: nothing uses what comes of them.)
            const X* src[XP];
            const W* wsrc[WP];
#pragma unroll
            for (int p = 0; p < XP; ++p) src[p] = xp + (int64_t)sh.rows[min(xrow + p * (kAdThreads / XU), n_rows - 1)] * P.ldx + xu + k_from;
#pragma unroll
            for (int p = 0; p < WP; ++p) wsrc[p] = wa + (int64_t)min(c0 + wrow + p * (kAdThreads / WU), r_all - 1) * P.a_row + wu + k_from;
            const auto fill = [&](int i, int slot) {
                unsigned char* xs = stage + slot * s1 + xrow * Z::xld + tid % XU * 16;
                unsigned char* ws = stage + slot * s1 + T * Z::xld + wrow * Z::ald + tid % WU * 16;
                const int k = i * KC, left = k_to - k_from - k;
                if (left >= KC && P.wide_x && P.wide_a) {
#pragma unroll
                    for (int p = 0; p < XP; ++p)
                        if (xrow + p * (kAdThreads / XU) < n_rows) ad_copy16(xs + p * (kAdThreads / XU) * Z::xld, src[p] + k);
#pragma unroll
                    for (int p = 0; p < WP; ++p)
                        if (wrow + p * (kAdThreads / WU) < 8 * nt) ad_copy16(ws + p * (kAdThreads / WU) * Z::ald, wsrc[p] + k);
                    return;
                }
#pragma unroll
                for (int p = 0; p < XP; ++p) ad_fill16(xs + p * (kAdThreads / XU) * Z::xld, src[p] + k, left - xu, P.wide_x);
#pragma unroll
                for (int p = 0; p < WP; ++p)
                    if (wrow + p * (kAdThreads / WU) < 8 * nt) ad_fill16(ws + p * (kAdThreads / WU) * Z::ald, wsrc[p] + k, left - wu, P.wide_a);
            };
            // NT groups of eight ranks (SOME: of which some may be missing; without a branch per group their products run side by side).  The tensor core takes
            // sixteen of one operand and eight of the other: rows and ranks, or, where there are few rows (FEW: up to eight), ranks and rows, which is half
            // the products and half the splitting.
            const auto products = [&](auto groups_of_8, auto some_missing, auto few_rows) {
                constexpr int NT = decltype(groups_of_8)::value;
                constexpr bool SOME = decltype(some_missing)::value, FEW = decltype(few_rows)::value;
                constexpr int G = FEW ? 2 : 1, NG = NT / G;  // groups of eight that a product takes
                float acc[NG][4];
#pragma unroll
                for (int j = 0; j < NG; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
                ad_pipeline<Z::stages>(count, fill, [&](int, int slot) {
#pragma unroll
                    for (int s = 0; s < KC / 16 / KS; ++s) {
                        if constexpr (Z::wide) {
                            // A lane has four consecutive k of every row; the products do not mind in which order the tensor core takes them, as long as both
                            // operands agree.
                            const int k = 16 * (ks + KS * s) + 4 * q;
                            const unsigned char* xs = stage + slot * s1 + (16 * mt + g) * Z::xld + k * 4;
                            const unsigned char* ws = stage + slot * s1 + T * Z::xld + g * Z::ald + k * 2;
                            uint32_t hi[2][4], lo[2][4];
#pragma unroll
                            for (int h = 0; h < (FEW ? 1 : 2); ++h) {
                                const float4 y = *reinterpret_cast<const float4*>(xs + 8 * h * Z::xld);
                                ad_split(y.x, hi[h][0], lo[h][0]);
                                ad_split(y.y, hi[h][1], lo[h][1]);
                                ad_split(y.z, hi[h][2], lo[h][2]);
                                ad_split(y.w, hi[h][3], lo[h][3]);
                            }
#pragma unroll
                            for (int j = 0; j < NG; ++j)
                                if (!SOME || G * j < nt) {
                                    uint32_t b[G][4];
#pragma unroll
                                    for (int h = 0; h < G; ++h) {
                                        const float4 v = ad_floats(*reinterpret_cast<const uint2*>(ws + 8 * (G * j + h) * Z::ald), (const W*)nullptr);
                                        b[h][0] = __float_as_uint(v.x), b[h][1] = __float_as_uint(v.y), b[h][2] = __float_as_uint(v.z), b[h][3] = __float_as_uint(v.w);
                                    }
                                    // The tensor core cuts its sums, always towards zero: sixteen k by themselves, which are then added with rounding (10240 k of
                                    // random numbers, 64 adapters: outputs 7.7e-7 off without this, 0.9e-7 with it).
                                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                    for (int p = 0; p < 2; ++p) {
                                        const auto& x = p ? hi : lo;
#pragma unroll
                                        for (int e = 0; e < 4; e += 2) {
                                            if constexpr (FEW)
                                                ad_mma_tf32(c, b[0][e], b[1][e], b[0][e + 1], b[1][e + 1], x[0][e], x[0][e + 1]);
                                            else
                                                ad_mma_tf32(c, x[0][e], x[1][e], x[0][e + 1], x[1][e + 1], b[0][e], b[0][e + 1]);
                                        }
                                    }
#pragma unroll
                                    for (int e = 0; e < 4; ++e) acc[j][e] += c[e];
                                }
                        } else {
                            // (this lane's row of the operands, and which of its two halves)
                            const uint32_t xm = smem_u32(stage + slot * s1 + (16 * mt + (lane & 15)) * Z::xld + (lane >> 4) * 16);
                            const uint32_t wm = smem_u32(stage + slot * s1 + T * Z::xld + ((lane & 7) + (lane >> 4) * 8) * Z::ald + (lane >> 3 & 1) * 16);
                            uint32_t y[4];
                            ad_ldm(y, xm + 32 * (ks + KS * s));
#pragma unroll
                            for (int j = 0; j < NT; j += 2)
                                if (!SOME || j < nt) {  // (a second one past the last rank: zeros or numbers that nothing uses)
                                    uint32_t b[4];
                                    ad_ldm(b, wm + 8 * j * Z::ald + 32 * (ks + KS * s));
                                    if constexpr (FEW) {
                                        ad_mma16(acc[j / 2], b[0], b[2], b[1], b[3], y[0], y[2], (const W*)nullptr);
                                    } else {
                                        ad_mma16(acc[j], y[0], y[1], y[2], y[3], b[0], b[1], (const W*)nullptr);
                                        ad_mma16(acc[j + 1], y[0], y[1], y[2], y[3], b[2], b[3], (const W*)nullptr);
                                    }
                                }
                        }
                    }
                });
                // the warps' sums meet: sums[ks][row][rank]
#pragma unroll
                for (int j = 0; j < NG; ++j)
                    if (G * j < nt) {
                        if constexpr (FEW) {
                            float* s0 = sums + ((ks * T + 2 * q) * kAdSumLd + 16 * j + g);
                            s0[0] = acc[j][0], s0[kAdSumLd] = acc[j][1];
                            s0[8] = acc[j][2], s0[kAdSumLd + 8] = acc[j][3];
                        } else {
                            float* s0 = sums + ((ks * T + 16 * mt + g) * kAdSumLd + 8 * j + 2 * q);
                            *reinterpret_cast<float2*>(s0) = make_float2(acc[j][0], acc[j][1]);
                            *reinterpret_cast<float2*>(s0 + 8 * kAdSumLd) = make_float2(acc[j][2], acc[j][3]);
                        }
                    }
            };
            const auto by_ranks = [&](auto few) {
                if (nt <= 2)
                    products(std::integral_constant<int, 2>(), std::false_type(), few);
                else if (Z::most_rank <= 32 || nt <= 4)
                    products(std::integral_constant<int, 4>(), std::false_type(), few);
                else if constexpr (Z::most_rank > 32) {
                    if (nt == 8)
                        products(std::integral_constant<int, 8>(), std::false_type(), few);
                    else
                        products(std::integral_constant<int, 8>(), std::true_type(), few);
                }
            };
            if (MT == 1 && n_rows <= 8)
                by_ranks(std::integral_constant<bool, MT == 1>());
            else
                by_ranks(std::false_type());
            __syncthreads();
            const int cols = (ranks + 15) / 16 * 16;  // (ranks behind the last one: zeros)
            for (int i = tid; i < T * cols / 4; i += kAdThreads) {
                const int row = i / (cols / 4), c = i % (cols / 4) * 4;
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c < ranks) {
#pragma unroll
                    for (int p = 0; p < KS; ++p) {
                        const float4 v = *reinterpret_cast<const float4*>(sums + (p * T + row) * kAdSumLd + c);
                        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                    }
                    if (c + 1 >= ranks) s.y = 0.f;
                    if (c + 2 >= ranks) s.z = 0.f;
                    if (c + 3 >= ranks) s.w = 0.f;
                }
                *reinterpret_cast<float4*>(part + row * cap + c0 + c) = s;
            }
        }
        // ---- the CTAs' parts meet, and become 16-bit operands
        const float scale = P.scales ? __ldg(P.scales + a) : 1.f;
        if (S > 1) {
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            __syncthreads();
        }
        constexpr int TPR = kAdThreads / T;  // threads of a row
        const int row = tid / TPR, c = tid % TPR;
        constexpr bool scaled = std::is_same<W, __half>::value;
        float most = 0.f;
        uint32_t small = ~0u;  // bits of the smallest that is not 0, times two, less one
        for (int i = 4 * c; i < r16; i += 4 * TPR) {
            float4 s = *reinterpret_cast<const float4*>(part + row * cap + i);
            if (S > 1) {
                s = make_float4(0.f, 0.f, 0.f, 0.f);
                const uint32_t at = smem_u32(part + row * cap + i);
                float4 v[kAdMaxCtas];
#pragma unroll
                for (int p = 0; p < kAdMaxCtas; ++p)
                    if (p < S) {
                        uint32_t from;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at), "r"(p));
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[p].x), "=f"(v[p].y), "=f"(v[p].z), "=f"(v[p].w) : "r"(from) : "memory");
                    }
#pragma unroll
                for (int p = 0; p < kAdMaxCtas; ++p)
                    if (p < S) s.x += v[p].x, s.y += v[p].y, s.z += v[p].z, s.w += v[p].w;
            }
            if (scaled)
                small = min(small, min(min(2 * __float_as_uint(s.x) - 1, 2 * __float_as_uint(s.y) - 1), min(2 * __float_as_uint(s.z) - 1, 2 * __float_as_uint(s.w) - 1)));
            most = fmaxf(most, fmaxf(fmaxf(fabsf(s.x), fabsf(s.y)), fmaxf(fabsf(s.z), fabsf(s.w))));
            *reinterpret_cast<float4*>(sums + row * cap + i) = s;
        }
#pragma unroll
        for (int o = TPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // fp16: relative to the power of two that brings the row's largest to 2^14 .. 2^15.  Two of them are 2^-24 of a value off, but no less than 2^-25.  (Beside an
        // infinity, which stays one, finite values are under 2^15 as well.)
        bool far = most > 0.f && most < INFINITY && !(most >= 0x1p-100f && most < 0x1p100f);
        float up = 1.f, down = scaled || most < INFINITY ? 1.f : 0.5f;
        if (scaled && most > 0.f && !far) {
            constexpr uint32_t below = Z::wide ? 20 : 23;
            const uint32_t e = __float_as_uint(most) >> 23;  // (27 .. 226, or 255)
            up = __uint_as_float((e - 14) << 23);
            down = __uint_as_float((268 - e) << 23);
            const uint32_t least = (e + 1 - below) << 23;
            if (__builtin_expect(small < 2 * least - 1 && most < INFINITY && row < n_rows, 0)) {
                far = S == 1;
                if (!far)
#pragma unroll 1
                    for (int i = 4 * c; i < r16; i += 4 * TPR)
#pragma unroll 1
                        for (int j = i; j < i + 4; ++j) {
                            if (2 * __float_as_uint(sums[row * cap + j]) - 1 >= 2 * least - 1) continue;
                            float m = 0.f;
#pragma unroll 4
                            for (int p = 0; p < S; ++p) {
                                uint32_t from;
                                float v;
                                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(smem_u32(part + row * cap + j)), "r"(p));
                                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
                                m = fmaxf(m, fabsf(v));
                            }
                            far |= __float_as_uint(m) < least;
                        }
            }
        }
        if (far && row < n_rows) sh.apart = 1;
        if (c == 0) sh.scale[row] = up * scale;
        for (int i = 4 * c; i < r16; i += 4 * TPR) {
            const float4 s = *reinterpret_cast<const float4*>(sums + row * cap + i);
            float f[4] = {s.x * down, s.y * down, s.z * down, s.w * down};
#pragma unroll
            for (int p = 0; p < pieces; ++p) {
                W h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[e] = ad_round<W>(f[e]);
                    const float b = ad_f32(h[e]);
                    f[e] = fabsf(b) == INFINITY ? 0.f : f[e] - b;
                }
                *reinterpret_cast<uint2*>(t16 + (p * T + row) * pld + i * 2) = *reinterpret_cast<const uint2*>(h);
            }
        }
        if (S > 1) {
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (nothing of the others is read from here on)
        }
    }
    __syncthreads();

    // ---- out = base + B t: this CTA's part of M, FB outputs and 64 ranks at a time through shared memory
    const int units = (P.M + 31) / 32, m_from = 32 * (int)((long long)units * rank / S), m_to = min(P.M, 32 * (int)((long long)units * (rank + 1) / S));
    const int chunks = max(1, (r16 + kAdChunk - 1) / kAdChunk), rc = min(r16, kAdChunk), wld = Z::wld(rc), s2 = Z::stage2(rc);
    const int count = (max(m_to - m_from, 0) + FB - 1) / FB * chunks;
    float t0 = r_all ? sh.scale[16 * mt + g] : 0.f, t1 = r_all ? sh.scale[16 * mt + g + 8] : 0.f;
    const bool have0 = 16 * mt + g < n_rows, have1 = 16 * mt + g + 8 < n_rows;
    X* o0 = op + (int64_t)sh.rows[min(16 * mt + g, n_rows - 1)] * P.ldout + m_from + FW * ks + 4 * q;  // of this stage
    X* o1 = op + (int64_t)sh.rows[min(16 * mt + g + 8, n_rows - 1)] * P.ldout + m_from + FW * ks + 4 * q;
    const W* wb = reinterpret_cast<const W*>(P.b) + (has ? a * P.b_slot : 0);
    // units of 16 bytes of a row of B, as a power of two
    const int lw = rc <= 8 ? 0 : rc <= 16 ? 1 : rc <= 32 ? 2 : 3, wu = tid & ((1 << lw) - 1), wrow = tid >> lw, wstep = kAdThreads >> lw;
    // output 4 x + 2 y + z of sixteen is row 8 y + 2 x + z: column 2 x + z of product y
    const int wat = (wrow & ~15) + (wrow >> 1 & 1) * 8 + (wrow >> 2 & 3) * 2 + (wrow & 1);
    constexpr int XN = 16 / (int)sizeof(X), BU = FB / XN, BP = T * BU / kAdThreads;
    const int bu = tid % BU * XN, brow = tid / BU;
    const W* wnext = wb + (int64_t)(m_from + wrow) * P.b_row + 8 * wu;  // of the next stage: they are begun in order
    const int64_t wrows = (int64_t)wstep * P.b_row;
    const X* bnext[BP];
#pragma unroll
    for (int p = 0; p < BP; ++p) bnext[p] = bp + (bp ? (int64_t)sh.rows[min(brow + p * (kAdThreads / BU), n_rows - 1)] * P.ldbase + m_from + bu : 0);
    const bool wide_in = P.wide_b && (!bp || P.wide_base);
    const auto fill = [&](int i, int slot) {
        unsigned char* ws = stage + slot * s2;
        unsigned char* bs = ws + FB * wld + brow * Z::bld + tid % BU * 16;
        const int fb = chunks == 1 ? i : i / chunks, ch = chunks == 1 ? 0 : i % chunks, left = m_to - m_from - fb * FB, r = ch * kAdChunk + 8 * wu;
        const bool whole = wide_in && left >= FB;
        if (r < r16) {
            const W* from = wnext + ch * kAdChunk;
            unsigned char* to = ws + wat * wld + wu * 16;
            const int bytes = max(0, min(8, r_all - r)) * 2;
#pragma unroll 2
            for (int f = wrow; f < FB; f += wstep) {
                if (whole)
                    ad_copy16(to, bytes ? from : wb, bytes);
                else
                    ad_fill16(to, from, f < left ? r_all - r : 0, P.wide_b);
                from += wrows;
                to += wstep * wld;
            }
        }
        if (ch == chunks - 1) {
            wnext += FB * P.b_row;
            if (bp)
#pragma unroll
                for (int p = 0; p < BP; ++p) {
                    if (whole) {
                        if (brow + p * (kAdThreads / BU) < n_rows) ad_copy16(bs + p * (kAdThreads / BU) * Z::bld, bnext[p]);
                    } else
                        ad_fill16(bs + p * (kAdThreads / BU) * Z::bld, bnext[p], left - bu, P.wide_base);
                    bnext[p] += FB;
                }
        }
    };
    const uint32_t wm = smem_u32(stage) + (FW * ks + (lane & 7) + (lane >> 4) * 8) * wld + (lane >> 3 & 1) * 16;
    const uint32_t tm = smem_u32(t16) + (16 * mt + (lane & 15)) * pld + (lane >> 4) * 16;
    // SK groups of sixteen ranks, whose operand of t a warp keeps (0: any number, read again; -1: t in fp32)
    const auto outputs = [&](auto groups_of_16) {
        constexpr int SK = decltype(groups_of_16)::value;
        uint32_t kept[SK > 0 ? SK : 1][pieces][4];
#pragma unroll
        for (int k = 0; k < SK; ++k)
#pragma unroll
            for (int p = 0; p < pieces; ++p) ad_ldm(kept[k][p], tm + p * T * pld + 32 * k);
        float acc[J][4];
        ad_pipeline<Z::stages>(count, fill, [&](int i, int slot) {
            const uint32_t ws = wm + slot * s2;
            const unsigned char* bs = stage + slot * s2 + FB * wld;
            const int fb = SK > 0 || chunks == 1 ? i : i / chunks, ch = SK > 0 || chunks == 1 ? 0 : i % chunks, steps = SK > 0 ? SK : min(kAdChunk, r16 - ch * kAdChunk) / 16;
            if (ch == 0)
#pragma unroll
                for (int j = 0; j < J; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            const uint32_t tp = tm + ch * kAdChunk * 2;
            if constexpr (SK < 0) {
                // (four consecutive ranks of every row, as in the first product)
                const float* tr = t32 + (16 * mt + g) * (cap + 8) + ch * kAdChunk + 4 * q;
                const unsigned char* wr = stage + slot * s2 + (FW * ks + g) * wld + 8 * q;
#pragma unroll 1
                for (int k = 0; k < steps; ++k) {
                    uint32_t hi[2][4], lo[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 y = *reinterpret_cast<const float4*>(tr + 8 * h * (cap + 8) + 16 * k);
                        ad_split(y.x, hi[h][0], lo[h][0]);
                        ad_split(y.y, hi[h][1], lo[h][1]);
                        ad_split(y.z, hi[h][2], lo[h][2]);
                        ad_split(y.w, hi[h][3], lo[h][3]);
                    }
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float4 v = ad_floats(*reinterpret_cast<const uint2*>(wr + 8 * j * wld + 32 * k), (const W*)nullptr);
                        const uint32_t b[4] = {__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)};
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            const auto& x = p ? hi : lo;
#pragma unroll
                            for (int e = 0; e < 4; e += 2) ad_mma_tf32(c, x[0][e], x[1][e], x[0][e + 1], x[1][e + 1], b[e], b[e + 1]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] += c[e];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < (SK < 0 ? 0 : SK ? SK : kAdChunk / 16); ++k)
                if (SK || k < steps) {
                    uint32_t w[J / 2][4];
#pragma unroll
                    for (int j = 0; j < J / 2; ++j) ad_ldm(w[j], ws + 16 * j * wld + 32 * k);
#pragma unroll
                    for (int p = pieces - 1; p >= 0; --p) {
                        uint32_t t[4];
                        if constexpr (SK)
                            t[0] = kept[k % (SK > 0 ? SK : 1)][p][0], t[1] = kept[k % (SK > 0 ? SK : 1)][p][1], t[2] = kept[k % (SK > 0 ? SK : 1)][p][2], t[3] = kept[k % (SK > 0 ? SK : 1)][p][3];
                        else
                            ad_ldm(t, tp + p * T * pld + 32 * k);
#pragma unroll
                        for (int j = 0; j < J; ++j) ad_mma16(acc[j], t[0], t[1], t[2], t[3], w[j / 2][j % 2 * 2], w[j / 2][j % 2 * 2 + 1], (const W*)nullptr);
                    }
                }
            if (ch == chunks - 1) {
                const int left = m_to - m_from - fb * FB - FW * ks - 4 * q;
                const bool whole = P.wide_out && m_from + (fb + 1) * FB <= m_to;
                const unsigned char* b0 = bs + (16 * mt + g) * Z::bld + (FW * ks + 4 * q) * (int)sizeof(X);
#pragma unroll
                for (int h = 0; h < FW / 16; ++h) {
                    // a lane has four neighbouring outputs of two rows
                    float4 v0 = make_float4(0.f, 0.f, 0.f, 0.f), v1 = v0;
                    if (bp) {
                        if constexpr (Z::wide) {
                            v0 = *reinterpret_cast<const float4*>(b0 + 64 * h), v1 = *reinterpret_cast<const float4*>(b0 + 8 * Z::bld + 64 * h);
                        } else {
                            v0 = ad_floats(*reinterpret_cast<const uint2*>(b0 + 32 * h), (const X*)nullptr);
                            v1 = ad_floats(*reinterpret_cast<const uint2*>(b0 + 8 * Z::bld + 32 * h), (const X*)nullptr);
                        }
                    }
                    if (r_all) {
                        v0 = make_float4(fmaf(t0, acc[2 * h][0], v0.x), fmaf(t0, acc[2 * h][1], v0.y), fmaf(t0, acc[2 * h + 1][0], v0.z), fmaf(t0, acc[2 * h + 1][1], v0.w));
                        v1 = make_float4(fmaf(t1, acc[2 * h][2], v1.x), fmaf(t1, acc[2 * h][3], v1.y), fmaf(t1, acc[2 * h + 1][2], v1.z), fmaf(t1, acc[2 * h + 1][3], v1.w));
                    }
                    if (whole) {
                        if (have0) ad_store4(o0 + 16 * h, v0);
                        if (have1) ad_store4(o1 + 16 * h, v1);
                    } else {
                        if (have0) ad_store4(o0 + 16 * h, v0, left - 16 * h, P.wide_out);
                        if (have1) ad_store4(o1 + 16 * h, v1, left - 16 * h, P.wide_out);
                    }
                }
                o0 += FB;
                o1 += FB;
            }
        });
    };
    const bool apart = r_all > 0 && sh.apart;
    if (r16 == 16 && !apart)
        outputs(std::integral_constant<int, 1>());
    else if (r16 == 32 && !apart)
        outputs(std::integral_constant<int, 2>());
    else if (Z::most_rank > 32 && r16 == 64 && !apart)
        outputs(std::integral_constant<int, (Z::most_rank > 32 ? 4 : 0)>());
    else if (!apart)
        outputs(std::integral_constant<int, 0>());
    else {  // t as it is, where its 16-bit numbers were
        for (int i = tid; i < T * r16 / 4; i += kAdThreads) {
            const int row = i / (r16 / 4), c = i % (r16 / 4) * 4;
            *reinterpret_cast<float4*>(t32 + row * (cap + 8) + c) = *reinterpret_cast<const float4*>(sums + row * cap + c);
        }
        t0 = t1 = P.scales ? __ldg(P.scales + a) : 1.f;
        __syncthreads();
        outputs(std::integral_constant<int, -1>());
    }
    if (r_all > 0 && S > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // no CTA leaves while its part may be read
    }
}

}  // namespace rsv
