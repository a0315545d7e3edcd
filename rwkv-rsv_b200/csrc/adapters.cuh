// Low-rank adapters of many requests at once, beside a projection that all rows share:
//   out[n] = base[n] + scale[a] B[a] (A[a] x[n]),  a = index[n]; rows with an index outside 0 .. slots - 1 have no adapter: out[n] = base[n].
//
// One launch, no work area.  A cluster of CTAs takes a tile: up to 16 MT rows of one adapter, wherever they lie.  Which ones follows from the indices
// alone: every cluster counts the rows per adapter, numbers the tiles adapter by adapter and gathers the rows of its own (of 4096 rows at a time, so that
// this stays short).  So an adapter is read once per tile, not once per row, and the host need not know the indices.
//   t = A x   the CTAs of the cluster split K, the warps of a CTA split it again; the partial sums meet in shared memory and then in the cluster's.
//   B t       the CTAs split M; every CTA has all of t.
// Both products run on the tensor cores with fp32 sums.  16-bit activations are operands as they are; fp32 ones are two tf32 numbers each, rounded to
// nearest (together 2^-24 off, as fp32 itself), and the 16-bit weights are exact in tf32.  t is two fp16 numbers per value, relative to the row's largest
// (2^-25 of it off), or two bf16 ones (2^-17; three, 2^-25, where out is fp32), so that B is an operand as it is.
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
    int wide_x, wide_a, wide_b, wide_out;  // four values at a time may be loaded (stored)
    int copies;                            // rows without adapter are written
};

constexpr int kAdThreads = 256;
constexpr int kAdWarps = kAdThreads / 32;
constexpr int kAdMaxRank = 256;
constexpr int kAdMaxSlots = 4096;
constexpr int kAdBlockRows = 4096;
constexpr int kAdMaxCtas = 8;
constexpr int kAdChunk = 64;  // ranks whose sums a warp holds at a time

template <typename X, typename W>
struct AdTypes {
    static constexpr bool wide = sizeof(X) == 4;                                                    // fp32 activations
    static constexpr int pieces = sizeof(X) == 4 && std::is_same<W, __nv_bfloat16>::value ? 3 : 2;  // 16-bit numbers for a value of t
};
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

// Four values from p on, of which the first n exist (the others are 0).
__device__ __forceinline__ float4 ad_load4(const float* p, int n, bool wide) {
    if (wide && n >= 4) return *reinterpret_cast<const float4*>(p);
    return make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
}
template <typename H>
__device__ __forceinline__ uint2 ad_load4(const H* p, int n, bool wide) {
    if (wide && n >= 4) return *reinterpret_cast<const uint2*>(p);
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
    uint2 v;
    v.x = (n > 0 ? (uint32_t)q[0] : 0u) | (n > 1 ? (uint32_t)q[1] << 16 : 0u);
    v.y = (n > 2 ? (uint32_t)q[2] : 0u) | (n > 3 ? (uint32_t)q[3] << 16 : 0u);
    return v;
}
__device__ __forceinline__ float ad_lo(uint32_t v, const __half*) { return __half2float(__ushort_as_half((unsigned short)v)); }
__device__ __forceinline__ float ad_hi(uint32_t v, const __half*) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
__device__ __forceinline__ float ad_lo(uint32_t v, const __nv_bfloat16*) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float ad_hi(uint32_t v, const __nv_bfloat16*) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ float4 ad_floats(const float4& v, const float*) { return v; }
template <typename H>
__device__ __forceinline__ float4 ad_floats(const uint2& v, const H* h) { return make_float4(ad_lo(v.x, h), ad_hi(v.x, h), ad_lo(v.y, h), ad_hi(v.y, h)); }
__device__ __forceinline__ void ad_store4(float* p, const float4& v, int n, bool wide) {
    if (wide && n >= 4) {
        *reinterpret_cast<float4*>(p) = v;
        return;
    }
    if (n > 0) p[0] = v.x;
    if (n > 1) p[1] = v.y;
    if (n > 2) p[2] = v.z;
    if (n > 3) p[3] = v.w;
}
template <typename H>
__device__ __forceinline__ void ad_store4(H* p, const float4& v, int n, bool wide) {
    const H h[4] = {ad_round<H>(v.x), ad_round<H>(v.y), ad_round<H>(v.z), ad_round<H>(v.w)};
    if (wide && n >= 4) {
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = h[i];
}

__device__ __forceinline__ uint32_t ad_tf32(float v) {
    uint32_t t;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(t) : "f"(v));
    return t;
}
// v as two tf32 numbers (an infinity has no rest)
__device__ __forceinline__ void ad_split(float v, uint32_t& hi, uint32_t& lo) {
    hi = ad_tf32(v);
    const float h = __uint_as_float(hi);
    lo = ad_tf32(fabsf(h) == INFINITY ? 0.f : v - h);
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

// Shared memory: rows | t, this CTA's part [16 MT][rank_cap] fp32 | t's pieces [pieces][16 MT][rank_cap + 8] | sums of the warps (before: counters of the adapters).
__host__ __device__ constexpr size_t ad_part_bytes(int T, int cap) { return (size_t)T * cap * 4; }
__host__ __device__ constexpr size_t ad_piece_bytes(int T, int cap, int pieces) { return (size_t)pieces * T * (cap + 8) * 2; }
constexpr int kAdSumLd = kAdChunk + 8;  // (rows eight banks apart)
constexpr size_t kAdSumBytes = (size_t)kAdWarps * 16 * kAdSumLd * 4;
constexpr int kAdMostCells = 8192;  // rows x rank_cap of a tile: t lies where the sums were
static_assert((kAdMaxSlots + 2) * 2 <= kAdSumBytes && kAdMostCells * 4 <= kAdSumBytes, "the counters lie where the sums go later, and t after them");
__host__ __device__ constexpr size_t ad_smem(int T, int cap, int pieces) { return 1024 + ad_part_bytes(T, cap) + ad_piece_bytes(T, cap, pieces) + kAdSumBytes; }

struct AdTile {
    int rows[64];
    float scale[64];  // 2^e of the row's t, times the adapter's scale
    int slot, n, wsum[kAdWarps];
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
    const int tid = threadIdx.x, groups = P.slots + 1;  // the last one: rows without adapter
    for (int i = tid; i < (groups + 1) / 2; i += kAdThreads) reinterpret_cast<uint32_t*>(cnt)[i] = 0;
    if (tid == 0) sh.slot = -1;
    __syncthreads();
    const int32_t* ix = P.index + first;
    const auto group = [&](int i) {
        const int a = ix[i];
        return a >= 0 && a < P.slots ? a : P.slots;
    };
    for (int i = tid; i < rows; i += kAdThreads) {
        const int g = group(i);
        atomicAdd(reinterpret_cast<uint32_t*>(cnt) + (g >> 1), g & 1 ? 65536u : 1u);  // (no counter passes 4096)
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
                sh.n = tile - at;
                break;
            }
            at += t;
        }
    __syncthreads();
    const int mine = sh.slot, skip = sh.n * T;
    __syncthreads();
    if (tid == 0) sh.n = min(T, (int)cnt[mine] - skip);
    const int each = (rows + kAdThreads - 1) / kAdThreads, i0 = min(tid * each, rows), i1 = min(i0 + each, rows);
    int n = 0;
    for (int i = i0; i < i1; ++i) n += group(i) == mine;
    int place = ad_before(n, sh.wsum, all) - skip;
    if (n && place < T && place + n > 0)
        for (int i = i0; i < i1; ++i)
            if (group(i) == mine) {
                if (place >= 0 && place < T) sh.rows[place] = first + i;
                ++place;
            }
    __syncthreads();
    return true;
}

template <typename X, typename W, int MT>
__global__ void __launch_bounds__(kAdThreads, 2) adapters_kernel(AdapterArgs P) {
    constexpr int T = 16 * MT, KS = kAdWarps / MT, pieces = AdTypes<X, W>::pieces;
    constexpr bool wide = AdTypes<X, W>::wide;
    extern __shared__ __align__(16) unsigned char ad_smem_bytes[];
    AdTile& sh = *reinterpret_cast<AdTile*>(ad_smem_bytes);
    const int cap = P.rank_cap, ld16 = cap + 8;
    float* part = reinterpret_cast<float*>(ad_smem_bytes + 1024);
    W* t16 = reinterpret_cast<W*>(ad_smem_bytes + 1024 + ad_part_bytes(T, cap));
    float* sums = reinterpret_cast<float*>(ad_smem_bytes + 1024 + ad_part_bytes(T, cap) + ad_piece_bytes(T, cap, pieces));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3, mt = warp % MT, ks = warp / MT;
    const int S = P.S, rank = S > 1 ? (int)ad_rank() : 0;
    const int job = (int)blockIdx.x / S, block = job / P.tiles, first = block * P.block_rows;
    if (!ad_find_tile<T>(P, first, min(P.block_rows, P.rows - first), job % P.tiles, sh, reinterpret_cast<unsigned short*>(sums))) return;  // (all CTAs of the cluster)
    const int n_rows = sh.n, a = sh.slot;
    const bool has = a < P.slots;
    const int r_all = !has ? 0 : P.ranks ? max(0, min(__ldg(P.ranks + a), P.max_rank)) : P.max_rank;
    const float scale = has && P.scales ? __ldg(P.scales + a) : 1.f;
    const X* xp = reinterpret_cast<const X*>(P.x);
    const X* bp = reinterpret_cast<const X*>(P.base);
    X* op = reinterpret_cast<X*>(P.out);
    // rows of this lane in the tile's products (rows past the last one repeat it and are not stored)
    const int64_t row0 = sh.rows[min(16 * mt + g, n_rows - 1)], row1 = sh.rows[min(16 * mt + g + 8, n_rows - 1)];

    if (r_all > 0) {
        // ---- t = A x: this CTA's part of K
        const int units = (P.K + 15) / 16, u0 = (int)((long long)units * rank / S), u1 = (int)((long long)units * (rank + 1) / S);
        const int v0 = u0 + (u1 - u0) * ks / KS, v1 = u0 + (u1 - u0) * (ks + 1) / KS;
        const X *x0 = xp + row0 * P.ldx, *x1 = xp + row1 * P.ldx;
        const W* wa = reinterpret_cast<const W*>(P.a) + a * P.a_slot;
#pragma unroll 1
        for (int c0 = 0; c0 < r_all; c0 += kAdChunk) {
            const int nt = (min(kAdChunk, r_all - c0) + 7) / 8;
            float acc[kAdChunk / 8][4];
#pragma unroll
            for (int j = 0; j < kAdChunk / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            const W* wr = wa + (int64_t)min(c0 + g, r_all - 1) * P.a_row;
#pragma unroll 1
            for (int v = v0; v < v1; ++v) {
                // A lane has four consecutive k of every row; the products do not mind in which order the tensor core takes them, as long as both operands agree.
                const int k = 16 * v + 4 * q, left = P.K - k;
                uint2 w[kAdChunk / 8];
#pragma unroll
                for (int j = 0; j < kAdChunk / 8; ++j)
                    if (j < nt) w[j] = c0 + 8 * j + g < r_all ? ad_load4(wr + (int64_t)8 * j * P.a_row + k, left, P.wide_a) : make_uint2(0u, 0u);
                const auto y0 = ad_load4(x0 + k, left, P.wide_x), y1 = ad_load4(x1 + k, left, P.wide_x);
                if constexpr (wide) {
                    const float f[2][4] = {{y0.x, y0.y, y0.z, y0.w}, {y1.x, y1.y, y1.z, y1.w}};
                    uint32_t hi[2][4], lo[2][4];
#pragma unroll
                    for (int i = 0; i < 8; ++i) ad_split(f[i >> 2][i & 3], hi[i >> 2][i & 3], lo[i >> 2][i & 3]);
#pragma unroll
                    for (int j = 0; j < kAdChunk / 8; ++j)
                        if (j < nt) {
                            const float4 b = ad_floats(w[j], (const W*)nullptr);
                            const uint32_t b0 = __float_as_uint(b.x), b1 = __float_as_uint(b.y), b2 = __float_as_uint(b.z), b3 = __float_as_uint(b.w);
                            ad_mma_tf32(acc[j], lo[0][0], lo[1][0], lo[0][1], lo[1][1], b0, b1);
                            ad_mma_tf32(acc[j], lo[0][2], lo[1][2], lo[0][3], lo[1][3], b2, b3);
                            ad_mma_tf32(acc[j], hi[0][0], hi[1][0], hi[0][1], hi[1][1], b0, b1);
                            ad_mma_tf32(acc[j], hi[0][2], hi[1][2], hi[0][3], hi[1][3], b2, b3);
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < kAdChunk / 8; ++j)
                        if (j < nt) ad_mma16(acc[j], y0.x, y1.x, y0.y, y1.y, w[j].x, w[j].y, (const W*)nullptr);
                }
            }
            // the warps' sums meet: sums[ks][row][rank]
            __syncthreads();  // (the counters, or the chunk before this one, have been read)
#pragma unroll
            for (int j = 0; j < kAdChunk / 8; ++j)
                if (j < nt) {
                    float* s0 = sums + ((ks * T + 16 * mt + g) * kAdSumLd + 8 * j + 2 * q);
                    *reinterpret_cast<float2*>(s0) = make_float2(acc[j][0], acc[j][1]);
                    *reinterpret_cast<float2*>(s0 + 8 * kAdSumLd) = make_float2(acc[j][2], acc[j][3]);
                }
            __syncthreads();
            const int cols = (min(kAdChunk, r_all - c0) + 15) / 16 * 16;  // (ranks behind the last one: zeros)
            for (int i = tid; i < T * cols / 4; i += kAdThreads) {
                const int row = i / (cols / 4), c = i % (cols / 4) * 4;
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c < 8 * nt)
#pragma unroll
                    for (int p = 0; p < KS; ++p) {
                        const float4 v = *reinterpret_cast<const float4*>(sums + (p * T + row) * kAdSumLd + c);
                        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                    }
                *reinterpret_cast<float4*>(part + row * cap + c0 + c) = s;
            }
        }
        // ---- the CTAs' parts meet, and become 16-bit operands
        if (S > 1) {
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            __syncthreads();
        }
        const int r16 = (r_all + 15) / 16 * 16;
        constexpr int TPR = kAdThreads / T;  // threads of a row
        {
            const int row = tid / TPR, c = tid % TPR;
            float most = 0.f;
            for (int i = 4 * c; i < r16; i += 4 * TPR) {
                float4 s = *reinterpret_cast<const float4*>(part + row * cap + i);
                if (S > 1) {
                    s = make_float4(0.f, 0.f, 0.f, 0.f);
                    const uint32_t at = smem_u32(part + row * cap + i);
#pragma unroll
                    for (int p = 0; p < kAdMaxCtas; ++p)
                        if (p < S) {
                            uint32_t from;
                            float4 v;
                            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at), "r"(p));
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(from) : "memory");
                            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                        }
                }
                most = fmaxf(most, fmaxf(fmaxf(fabsf(s.x), fabsf(s.y)), fmaxf(fabsf(s.z), fabsf(s.w))));
                *reinterpret_cast<float4*>(sums + row * cap + i) = s;
            }
#pragma unroll
            for (int o = TPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            // fp16: relative to a power of two from the row's largest on
            float up = 1.f, down = 1.f;
            if (std::is_same<W, __half>::value && most > 0.f && most < INFINITY) {
                const int e = min(max((int)(__float_as_uint(most) >> 23) - 126, -120), 126);
                up = __uint_as_float((uint32_t)(127 + e) << 23);
                down = __uint_as_float((uint32_t)(127 - e) << 23);
            }
            if (c == 0) sh.scale[row] = up * scale;
            __syncwarp();
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
                    *reinterpret_cast<uint2*>(t16 + (size_t)(p * T + row) * ld16 + i) = *reinterpret_cast<const uint2*>(h);
                }
            }
        }
        __syncthreads();
        if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (nothing of the others is read from here on)
    }

    // ---- out = base + B t: this CTA's part of M, 32 outputs at a time; an output's place in a product's columns is chosen so that a lane has four neighbours
    const int units = (P.M + 31) / 32, u0 = (int)((long long)units * rank / S), u1 = (int)((long long)units * (rank + 1) / S), ksteps = (r_all + 15) / 16;
    const float s0 = r_all ? sh.scale[16 * mt + g] : 0.f, s1 = r_all ? sh.scale[16 * mt + g + 8] : 0.f;
    const bool have0 = 16 * mt + g < n_rows, have1 = 16 * mt + g + 8 < n_rows;
    const W* wb = reinterpret_cast<const W*>(P.b) + (has ? a * P.b_slot : 0);
#pragma unroll 1
    for (int u = u0 + ks; u < u1; u += KS) {
        const int m = 32 * u;
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        float4 b[2][2];  // [row][half]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int f = m + 16 * h + 4 * q, left = P.M - f;
            b[0][h] = bp && have0 && left > 0 ? ad_floats(ad_load4(bp + row0 * P.ldbase + f, left, P.wide_out), (const X*)nullptr) : make_float4(0.f, 0.f, 0.f, 0.f);
            b[1][h] = bp && have1 && left > 0 ? ad_floats(ad_load4(bp + row1 * P.ldbase + f, left, P.wide_out), (const X*)nullptr) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll 2
        for (int k = 0; k < ksteps; ++k) {
            const int r = 16 * k + 4 * q, left = r_all - r;
            uint2 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int f = m + 16 * (j >> 1) + 4 * (g >> 1) + 2 * (j & 1) + (g & 1);
                w[j] = f < P.M ? ad_load4(wb + (int64_t)f * P.b_row + r, left, P.wide_b) : make_uint2(0u, 0u);
            }
#pragma unroll
            for (int p = pieces - 1; p >= 0; --p) {
                const W* t0 = t16 + (size_t)(p * T + 16 * mt + g) * ld16 + r;
                const uint2 a0 = *reinterpret_cast<const uint2*>(t0), a1 = *reinterpret_cast<const uint2*>(t0 + 8 * ld16);
#pragma unroll
                for (int j = 0; j < 4; ++j) ad_mma16(acc[j], a0.x, a1.x, a0.y, a1.y, w[j].x, w[j].y, (const W*)nullptr);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int f = m + 16 * h + 4 * q, left = P.M - f;
            float4 v0 = b[0][h], v1 = b[1][h];
            if (r_all) {
                v0 = make_float4(fmaf(s0, acc[2 * h][0], v0.x), fmaf(s0, acc[2 * h][1], v0.y), fmaf(s0, acc[2 * h + 1][0], v0.z), fmaf(s0, acc[2 * h + 1][1], v0.w));
                v1 = make_float4(fmaf(s1, acc[2 * h][2], v1.x), fmaf(s1, acc[2 * h][3], v1.y), fmaf(s1, acc[2 * h + 1][2], v1.z), fmaf(s1, acc[2 * h + 1][3], v1.w));
            }
            if (have0 && left > 0) ad_store4(op + row0 * P.ldout + f, v0, left, P.wide_out);
            if (have1 && left > 0) ad_store4(op + row1 * P.ldout + f, v1, left, P.wide_out);
        }
    }
    if (r_all > 0 && S > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // no CTA leaves while its part may be read
    }
}

}  // namespace rsv
