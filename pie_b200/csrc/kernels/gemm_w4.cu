// Products with 4-bit weights: y[M, N] = x[M, K] * W[N, K]^T, W[n, k] = s[n, k / G] * v(q[n, k]), with a 16-bit scale s per row and
// group of G = 32, 64 or 128 columns and a code q of 4 bits: v(q) = q - 8, q - z[n, k / G], or the e2m1 number q stands for.
//
// Layout (ops/w4.py writes it once, when a weight is loaded): codes lie in tiles of 16 rows x 64 columns, 512 bytes, in the order [128
// rows][64 columns][row tile], so that 128 rows of any range of columns are one piece of memory. A tile is the A operand of four
// m16n8k16 MMAs as the lanes hold it: lane 4 g + t has 16 bytes, word j of them for columns 32 (j >> 1) + 8 t + 4 (j & 1) .. + 3 of rows g
// (nibbles 0, 4, 1, 5; e2m1: 0, 1, 2, 3) and g + 8 (nibbles 2, 6, 3, 7; e2m1: 4, 5, 6, 7). A load of a tile is so one 16-byte load
// per lane, all of it used. Scales and zero points lie as [128 rows][group][row tile][8] pairs (row g, row g + 8). Scales are fp16,
// multiplied by a power of two per row that brings the row's largest to [2^14, 2^15), or for e2m1 [2^10, 2^11); `factor` undoes it.
// bf16 and fp16 scales are so held exactly down to 2^-24 of the row's largest; smaller ones lose bits, and below 2^-39 of it (e2m1: 2^-35) they
// are zero. Rows are padded to 128, columns to 64, with codes of value zero and scales of zero.
//
// Counterpart of the reference's W4A16 products (driver/cuda/src/kernels/dequant_wna16.cu and its mma.sync GEMM).
#include <atomic>

#include "gemm_common.cuh"

namespace pie {

// A packed weight, or `experts` of them one after the other (ops/w4.py has the same struct).
struct W4Weight {
    const uint4* codes;
    const uint32_t* scale;       // two fp16 scales a word
    const uint16_t* zero;        // two zero points a word, or null: 8
    const float* factor;         // [experts][panels * 128]
    int experts, n, k, group;
    int fp4;                     // codes are e2m1 and not integers

    __host__ __device__ int row_tiles() const { return (n + 15) >> 4; }
    __host__ __device__ int panels() const { return (n + 127) >> 7; }             // of 128 rows
    __host__ __device__ int blocks() const { return (k + 63) >> 6; }
    __host__ __device__ int groups() const { return group == 128 ? k >> 7 : blocks() * (64 / group); }
};

enum W4Kind : int { W4_INT = 0, W4_ZERO = 1, W4_FP4 = 2 };
static inline int w4_kind(const W4Weight& w) { return w.fp4 ? W4_FP4 : w.zero ? W4_ZERO : W4_INT; }

// Pair i of a word of codes as two bf16, exactly, times W4_UNIT<KIND>. Integers: the four bits at the bottom of a bf16, or four bits above
// them, are the subnormal number q 2^-133 or q 2^-129 (exponent fields 0 and 1 have one spacing), so two ands and a shift by 8 for the other
// two pairs are all the bit work; `zero` = -z / 64, twice, and a multiplication by 2^127 or 2^123 make it (q - z) / 64. e2m1: a byte is a pair and
// the machine converts it to fp16.
template <int KIND>
constexpr float W4_UNIT = KIND == W4_FP4 ? 1.f : 64.f;
__device__ __forceinline__ bf162 bf162_bits(uint32_t v) { return *reinterpret_cast<const bf162*>(&v); }
__device__ __forceinline__ __half2 half2_bits(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
// A word's bytes, two e2m1 numbers each, as fp16.
__device__ __forceinline__ void e2m1_pairs(uint32_t word, uint32_t (&r)[4]) {
    asm("{\n.reg .b8 b, c, d, e;\nmov.b32 {b, c, d, e}, %4;\ncvt.rn.f16x2.e2m1x2 %0, b;\ncvt.rn.f16x2.e2m1x2 %1, c;\n"
        "cvt.rn.f16x2.e2m1x2 %2, d;\ncvt.rn.f16x2.e2m1x2 %3, e;\n}\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(word));
}
__device__ __forceinline__ bf162 w4_pair(uint32_t word, int i, bf162 zero) {
    const uint32_t v = (i < 2 ? word : word >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
    return __hfma2(bf162_bits(v), bf162_bits(i & 1 ? 0x7d007d00u : 0x7f007f00u), zero);
}
// -z / 64, twice, of byte i of `z` (row g's zero point, row g + 8's): the byte is the number z 2^-133.
__device__ __forceinline__ bf162 w4_zero_of(uint32_t z, int i) {
    return __hmul2(bf162_bits(__byte_perm(z, 0u, i ? 0x4141 : 0x4040)), bf162_bits(0xff00ff00u));
}
// The four pairs of a word as operands of an MMA: bf16, of e2m1 fp16. z0, z1: `zero` of row g and row g + 8.
template <int KIND>
__device__ __forceinline__ void w4_pairs(uint32_t word, bf162 z0, bf162 z1, uint32_t (&r)[4]) {
    if (KIND == W4_FP4) return e2m1_pairs(word, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf162 v = w4_pair(word, i, i < 2 ? z0 : z1);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
__device__ __forceinline__ float2 w4_scales(uint32_t word) { return __half22float2(*reinterpret_cast<const __half2*>(&word)); }

// ------------------------------------------------------------------ expansion
// out[e][n][k] = bf16(s v(q)): the product is exact in 32 bits, so a weight is rounded once. One warp per tile of codes. Bound by the
// bytes it writes.
template <int KIND>
__global__ void __launch_bounds__(256) w4_expand_kernel(const W4Weight w, bf16* __restrict__ out) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int ps = w.panels(), kbs = w.blocks(), groups = w.groups();
    const long tiles = (long)w.experts * ps * kbs * 8;
    for (long tile = (long)blockIdx.x * 8 + (threadIdx.x >> 5); tile < tiles; tile += (long)gridDim.x * 8) {
        const long line = (tile >> 3) / kbs;                   // panel, counted over all experts
        const int kb = (int)((tile >> 3) - line * kbs), rt = (int)(line % ps) * 8 + (int)(tile & 7);
        const int left = w.n - rt * 16;                        // rows of the tile that exist
        if (left <= 0) continue;
        const uint4 c = w.codes[tile * 32 + lane];
        const long row = line / ps * w.n + rt * 16 + g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k0 = kb * 64 + (j >> 1) * 32 + t * 8 + (j & 1) * 4;
            if (k0 >= w.k) break;
            const long at = ((line * groups + k0 / w.group) * 8 + (tile & 7)) * 8 + g;
            const float2 s = w4_scales(w.scale[at]);
            const int z = KIND == W4_ZERO ? w.zero[at] : 0x0808;
            uint32_t v[4];
            w4_pairs<KIND>(j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w, w4_zero_of(z, 0), w4_zero_of(z, 1), v);
            auto value = [&](int i) { return KIND == W4_FP4 ? __half22float2(half2_bits(v[i])) : __bfloat1622float2(bf162_bits(v[i])); };
#pragma unroll
            for (int h = 0; h < 2; ++h) {                      // row g, row g + 8
                if (g + 8 * h >= left) break;
                const float2 a = value(2 * h), b = value(2 * h + 1);
                const float f = (h ? s.y : s.x) * w.factor[line * 128 + (tile & 7) * 16 + g + 8 * h] * W4_UNIT<KIND>;
                const bf162 o[2] = {__floats2bfloat162_rn(a.x * f, a.y * f), __floats2bfloat162_rn(b.x * f, b.y * f)};
                *reinterpret_cast<uint2*>(out + (row + 8 * h) * w.k + k0) = *reinterpret_cast<const uint2*>(o);
            }
        }
    }
}

// ------------------------------------------------------------------ few rows
// A CTA takes some row tiles and a share of K, a warp a row tile and every so many blocks of that: codes go from memory to the MMA's A
// registers, the batch's columns (eight at a time) from shared memory, where the CTA's share of them is brought first. Codes are exact in
// bf16, so a group's sum is of exact products; the scale is applied to it in 32 bits and no weight is rounded. The shares of K meet in
// shared memory, those of a cluster's CTAs in distributed shared memory, in order. Bound by the codes' latency (ncu: 39 % of DRAM, ALUs 40 %, warps
// wait for loads): 1 row through 28672 x 4096 15.0 us, 4.1 TB/s; through 4096 x 14336 7.9 us, 3.9 TB/s; 8 rows 17.9 and 9.0.

// bf16 operands, of e2m1 weights fp16.
template <int KIND>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (KIND == W4_FP4)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[2]), "r"(a[1]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[2]), "r"(a[1]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// Addresses and size multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// Waits until a copy is done, of a kernel that ends after a wait which ran out; itself limited.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!sm100::mbar_try_wait(bar, parity))
        if (clock64() - t0 > 200000000ll) return;
}

// Shared memory of a CTA: the batch's share (rows 64 bytes apart from a multiple of 128, so that two rows' pieces are in different
// banks) behind a barrier and the rows' largest values, the warps' sums as [warp][column][16 rows and 4 of padding], the cluster's as
// [CTA][column][feature], the rows' factors.
constexpr int W4R_BATCH = 150 * 1024;         // most of the batch in a CTA
constexpr int W4R_PAD = 20, W4R_HEAD = 16 + 32 * 4;
__host__ __device__ constexpr int w4r_row_bytes(int blocks) { return blocks * 128 + 64; }
__host__ __device__ constexpr int w4r_smem(int M, int blocks, int NT, int features, int ctas) {
    return W4R_HEAD + M * w4r_row_bytes(blocks) + 8 * NT * 8 * W4R_PAD * 4 + (ctas > 1 ? NT * 8 * features * 4 : 0) + features * 4;
}

// The batch's rows in shared memory, in place from bf16 to fp16, each times a power of two that brings its largest value to [2^14, 2^15)
// (a bf16 value keeps all its bits down to 2^-29 of that): e2m1 weights are fp16 by one instruction a pair, and six to bf16 would be what
// bounds the product. tops: the bits of the rows' largest values, zero before; all threads call. (A row with an infinity or NaN has
// nothing else in its results: what its other values become is of no matter.)
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }      // -126 .. 127
__device__ __forceinline__ int w4_row_exp(uint32_t top) { return top ? max(-126, min(126, 14 - ((int)(top >> 7) - 127))) : 0; }
__device__ __forceinline__ void w4_batch_fp16(uint8_t* batch, int row_bytes, int rows, int vecs, uint32_t* tops) {
    const int per_row = 3 - min(3, 31 - __clz(rows)), warp = threadIdx.x >> 5;        // 2^per_row of the eight warps take a row
    const int first = threadIdx.x & ((32 << per_row) - 1), step = 32 << per_row;
    for (int row = warp >> per_row; row < rows; row += 8 >> per_row) {
        uint32_t most = 0;
        for (int i = first; i < vecs; i += step) {
            const uint4 v = *reinterpret_cast<const uint4*>(batch + row * row_bytes + i * 16);
            most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        }
        most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
        if ((threadIdx.x & 31) == 0 && most) atomicMax(tops + row, most);
    }
    __syncthreads();
    for (int row = warp >> per_row; row < rows; row += 8 >> per_row) {
        const float f = exp2_int(w4_row_exp(tops[row]));
        auto pair = [&](uint32_t v) {
            const __half2 h = __floats2half2_rn(__uint_as_float(v << 16) * f, __uint_as_float(v & 0xffff0000u) * f);
            return *reinterpret_cast<const uint32_t*>(&h);
        };
        for (int i = first; i < vecs; i += step) {
            uint4* at = reinterpret_cast<uint4*>(batch + row * row_bytes + i * 16);
            const uint4 v = *at;
            *at = make_uint4(pair(v.x), pair(v.y), pair(v.z), pair(v.w));
        }
    }
    __syncthreads();
}

template <int GROUP>
constexpr int W4R_UNIT = GROUP == 128 ? 2 : 1;                    // blocks of 64 columns per unit of work: whole groups
template <int GROUP>
constexpr int W4R_SETS = GROUP == 32 ? 2 : 1;                     // scales per unit

// acc += a unit's codes times NT tiles of the batch's columns, which lie at xr.
template <int KIND, int GROUP, int NT>
__device__ __forceinline__ void w4_unit(const uint4 (&c)[W4R_UNIT<GROUP>], const uint32_t (&s)[W4R_SETS<GROUP>],
                                        const uint16_t (&z)[W4R_SETS<GROUP>], const uint8_t* const (&xr)[NT], float (&acc)[NT][4]) {
    constexpr int SETS = W4R_SETS<GROUP>, HALVES = W4R_UNIT<GROUP> * 2 / SETS;     // of 32 columns, per group
#pragma unroll
    for (int u = 0; u < SETS; ++u) {
        float sum[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[i][j] = 0.f;
        const int zw = KIND == W4_ZERO ? z[u] : 0x0808;
        const bf162 z0 = w4_zero_of(zw, 0), z1 = w4_zero_of(zw, 1);
#pragma unroll
        for (int h = u * HALVES; h < (u + 1) * HALVES; ++h) {
            uint4 b[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) b[i] = *reinterpret_cast<const uint4*>(xr[i] + h * 64);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4& v = c[h >> 1];
                const uint32_t word = h & 1 ? (j ? v.w : v.z) : (j ? v.y : v.x);
                uint32_t a[4];
                w4_pairs<KIND>(word, z0, z1, a);
#pragma unroll
                for (int i = 0; i < NT; ++i) mma_16816<KIND>(sum[i], a, j ? b[i].z : b[i].x, j ? b[i].w : b[i].y);
            }
        }
        const float2 f = w4_scales(s[u]);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            acc[i][0] = fmaf(f.x, sum[i][0], acc[i][0]);
            acc[i][1] = fmaf(f.x, sum[i][1], acc[i][1]);
            acc[i][2] = fmaf(f.y, sum[i][2], acc[i][2]);
            acc[i][3] = fmaf(f.y, sum[i][3], acc[i][3]);
        }
    }
}

// Sums of two rows of a batch in fp16 (columns of the MMA's tile), back to what the rows were.
__device__ __forceinline__ void w4_unscale(float (&acc)[4], const uint32_t* tops) {
    const float f0 = exp2_int(-w4_row_exp(tops[0])), f1 = exp2_int(-w4_row_exp(tops[1]));
    acc[0] *= f0; acc[1] *= f1; acc[2] *= f0; acc[3] *= f1;
}

// NT tiles of 8 batch rows, RESIDENT CTAs per SM. wk_shift: the block's eight warps are 2^wk_shift to a row tile, taking its units (a block
// of 64 columns, or two for groups of 128) in turn; 2^ct_shift CTAs (a cluster) share a tile's K.
template <int KIND, int GROUP, int NT, int RESIDENT>
__global__ void __launch_bounds__(256, RESIDENT)
w4_rows_kernel(const W4Weight w, const bf16* x, int ldx, bf16* C, int ldc, const bf16* R, int ldr, int M, int epi, int wk_shift,
               int ct_shift, int* status) {
    using namespace sm100;
    constexpr int UNIT = W4R_UNIT<GROUP>, SETS = W4R_SETS<GROUP>;
    constexpr int D = (RESIDENT == 2 && NT <= 2 ? 8 : 4) / UNIT;  // units on their way per lane
    extern __shared__ __align__(128) uint8_t rows_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = 1 << wk_shift, wr_shift = 3 - wk_shift, ctas = 1 << ct_shift, kbs = w.blocks(), groups = w.groups();
    const int rank = blockIdx.x & (ctas - 1), tile0 = (int)(blockIdx.x >> ct_shift) << wr_shift;
    const int units = kbs / UNIT, share = warp & (wk - 1);
    const int u0 = units * rank >> ct_shift, c_units = (units * (rank + 1) >> ct_shift) - u0;
    const int rt = min(tile0 + (warp >> wk_shift), w.panels() * 8 - 1);                     // rows past the last are not stored
    const uint4* codes = w.codes + (((size_t)(rt >> 3) * kbs + (u0 + share) * UNIT) * 8 + (rt & 7)) * 32 + lane;
    const size_t at = (((size_t)(rt >> 3) * groups + (u0 + share) * SETS) * 8 + (rt & 7)) * 8 + g;
    const uint32_t* scale = w.scale + at;
    const uint16_t* zero = w.zero + at;
    const int code_step = wk * UNIT * 256, set_step = wk * SETS * 64, x_step = wk * UNIT * 128;

    pdl_trigger();
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    uint4 c[D][UNIT];
    uint32_t s[D][SETS];
    uint16_t z[D][SETS];
    auto fetch = [&](int d) {                           // the unit that the pointers are at, and on
#pragma unroll
        for (int v = 0; v < UNIT; ++v) c[d][v] = ld_stream(codes + v * 256);
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            s[d][u] = __ldg(scale + u * 64);
            if (KIND == W4_ZERO) z[d][u] = __ldg(zero + u * 64);
        }
        codes += code_step;
        scale += set_step;
        zero += set_step;
    };
    int left = (c_units - share + wk - 1) >> wk_shift;  // units of this warp
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (d < left) fetch(d);

    const int features = 16 << wr_shift, row_bytes = w4r_row_bytes((units + ctas - 1 >> ct_shift) * UNIT);
    uint32_t* tops = reinterpret_cast<uint32_t*>(rows_smem + 16);
    uint8_t* batch = rows_smem + W4R_HEAD;
    float* parts = reinterpret_cast<float*>(batch + M * row_bytes);
    float* far = parts + 8 * NT * 8 * W4R_PAD;
    float* factors = far + (ctas > 1 ? NT * 8 * features : 0);
    const uint32_t bar = smem_addr(rows_smem);
    // The batch's rows: a copy each, of the columns that exist; the rest of the last block is zero.
    const int k0 = u0 * UNIT * 64, have = min(c_units * UNIT * 64, w.k - k0);
    if (KIND == W4_FP4 && threadIdx.x < NT * 8) tops[threadIdx.x] = 0;
    if (threadIdx.x < features) factors[threadIdx.x] = w.factor[tile0 * 16 + threadIdx.x];
    if (have < c_units * UNIT * 64 && threadIdx.x < 4 * M)
        *reinterpret_cast<uint4*>(batch + (threadIdx.x >> 2) * row_bytes + have * 2 + (threadIdx.x & 3) * 16) = make_uint4(0u, 0u, 0u, 0u);
    if (warp == 0) {
        if (lane == 0) {
            mbar_init(bar, 1);
            fence_barrier_init();
            fence_proxy_async();
            mbar_arrive_expect_tx(bar, M * have * 2);
        }
        __syncwarp();
        pdl_wait();                                     // the weights depend on nothing, the rows do
        for (int row = lane; row < M; row += 32) bulk_load(smem_addr(batch) + row * row_bytes, x + (size_t)row * ldx + k0, have * 2, bar);
    }
    __syncthreads();
    pdl_wait();                                         // outputs and residual may still be in use
    // a wait that runs out leaves numbers that are wrong and an error for the host
    if (!mbar_wait(bar, 0, status, PIE_ERR_WAIT_TMA)) drain(bar, 0);
    if (KIND == W4_FP4) w4_batch_fp16(batch, row_bytes, M, have >> 3, tops);
    __syncwarp();                                       // lanes may leave the wait one by one; an MMA is all of theirs
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    // columns past the batch's last are computed of its last row and not stored
    const uint8_t* xr[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) xr[i] = batch + min(i * 8 + g, M - 1) * row_bytes + share * UNIT * 128 + t * 16;

    auto unit = [&](int d) {
        w4_unit<KIND, GROUP, NT>(c[d], s[d], z[d], xr, acc);
#pragma unroll
        for (int i = 0; i < NT; ++i) xr[i] += x_step;
    };
    for (; left >= 2 * D; left -= D) {                  // D units here, and D more on their way
#pragma unroll
        for (int d = 0; d < D; ++d) {
            unit(d);
            fetch(d);
        }
    }
    for (; left > 0; left -= D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (d >= left) break;
            unit(d);
            if (D + d < left) fetch(d);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        if (KIND == W4_FP4) w4_unscale(acc[i], tops + i * 8 + 2 * t);
        float* at = parts + (warp * NT * 8 + i * 8 + 2 * t) * W4R_PAD + g;
        at[0] = acc[i][0];
        at[W4R_PAD] = acc[i][1];
        at[8] = acc[i][2];
        at[W4R_PAD + 8] = acc[i][3];
    }
    __syncthreads();
    // four features r .. of this CTA's sums for one row of the batch
    auto here = [&](int r, int col) {
        const float* at = parts + (((r >> 4) << wk_shift) * NT * 8 + col) * W4R_PAD + (r & 15);
        float4 v = *reinterpret_cast<const float4*>(at);
        for (int k = 1; k < wk; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(at + k * NT * 8 * W4R_PAD);
            v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
        }
        return v;
    };
    // features that this CTA stores, four or more
    const int mine_shift = 4 + wr_shift - ct_shift, mine = 1 << mine_shift, first = rank << mine_shift;
    if (ctas > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");              // all CTAs have started
        const uint32_t far_at = smem_addr(far) + rank * NT * 8 * mine * 4;
        for (int i = threadIdx.x; i < M << (2 + wr_shift); i += 256) {
            const int r = (i & (features / 4 - 1)) * 4, col = i >> (2 + wr_shift);
            const float4 v = here(r, col);
            st_cluster_v4(map_to_cta(far_at + ((col << mine_shift) + (r & (mine - 1))) * 4, r >> mine_shift), v.x, v.y, v.z, v.w);
        }
        __syncwarp();                                   // some lanes have a turn more
        cluster_sync_all();
    }
    const bool glu = epi == EPI_SWIGLU || epi == EPI_GEGLU;
    const int cols = glu ? w.n >> 1 : w.n;
    for (int i = threadIdx.x; i < M << (mine_shift - 2); i += 256) {
        const int r = (i & (mine / 4 - 1)) * 4, col = i >> (mine_shift - 2), f0 = tile0 * 16 + first + r;
        if (f0 >= w.n) continue;
        float4 v;
        if (ctas > 1) {
            const float* at = far + (col << mine_shift) + r;
            v = *reinterpret_cast<const float4*>(at);
            for (int k = 1; k < ctas; ++k) {
                const float4 y = *reinterpret_cast<const float4*>(at + (k * NT * 8 << mine_shift));
                v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
            }
        } else v = here(r, col);
        const float4 f = *reinterpret_cast<const float4*>(factors + first + r);
        v.x *= f.x * W4_UNIT<KIND>; v.y *= f.y * W4_UNIT<KIND>; v.z *= f.z * W4_UNIT<KIND>; v.w *= f.w * W4_UNIT<KIND>;
        if (glu) {
            const float a = epi == EPI_SWIGLU ? glu_value<EPI_SWIGLU>(v.x, v.y, 0.f) : glu_value<EPI_GEGLU>(v.x, v.y, 0.f);
            const float b = epi == EPI_SWIGLU ? glu_value<EPI_SWIGLU>(v.z, v.w, 0.f) : glu_value<EPI_GEGLU>(v.z, v.w, 0.f);
            *reinterpret_cast<bf162*>(C + (size_t)col * ldc + (f0 >> 1)) = __floats2bfloat162_rn(a, b);
        } else {
            if (epi == EPI_RESIDUAL) {
                const uint2 raw = *reinterpret_cast<const uint2*>(R + (size_t)col * ldr + f0);
                const float2 a = __bfloat1622float2(bf162_bits(raw.x)), b = __bfloat1622float2(bf162_bits(raw.y));
                v.x += a.x; v.y += a.y; v.z += b.x; v.w += b.y;
            }
            const bf162 o[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
            *reinterpret_cast<uint2*>(C + (size_t)col * ldc + f0) = *reinterpret_cast<const uint2*>(o);
        }
    }
}

// A sorted batch's tiles (as in gemm_grouped.cu), and the rows that one of them stands for.
struct W4Item {
    int row0, rows, expert;
};
struct W4Tiles {
    const int *expert, *list;
    int max_mtiles, experts;
    __device__ __forceinline__ int count() const { return list ? min(list[0], max_mtiles) : max_mtiles; }
    __device__ __forceinline__ W4Item at(int i) const {
        const int entry = list ? list[1 + i] : (i << 9 | GEMM_BM), tile = entry >> 9;
        const int e = (unsigned)tile < (unsigned)max_mtiles ? expert[tile] : -1;
        const int rows = min(min(entry & 511, 2 * GEMM_BM), (max_mtiles - tile) * GEMM_BM);
        return W4Item{tile * GEMM_BM, (unsigned)e < (unsigned)experts ? max(0, rows) : 0, e};
    }
};

// ------------------------------------------------------------------ few rows of many experts
// As above, for a sorted batch whose experts have a few rows each (a decode step): an item is up to eight rows of an expert, and the items'
// row tiles are dealt out to the CTAs of a resident grid in equal runs, so that a CTA mostly stays with one item's rows. 2^wk_shift warps
// share a row tile's K, by a rule on the number of row tiles, which the device alone knows; their sums meet in shared memory, one barrier
// per step, the next step's first codes being on their way. Bound by the latency of the codes, the scheduler's slots next: two CTAs per SM
// with eight units per lane on their way 44 us (64 tokens of 8 of 128 experts of 1536 x 2048), three with four 50, four with four 46, one with
// sixteen 53.
__host__ __device__ constexpr int w4e_smem(int blocks) { return W4R_HEAD + 8 * w4r_row_bytes(blocks) + 2 * 64 * W4R_PAD * 4; }

constexpr int W4E_STEPS = 4;
template <int KIND, int GROUP>
__global__ void __launch_bounds__(256, 2)
w4_experts_kernel(const W4Weight w, const bf16* x, int ldx, bf16* C, int ldc, const W4Tiles tiles, int epi, int* status) {
    using namespace sm100;
    constexpr int UNIT = W4R_UNIT<GROUP>, SETS = W4R_SETS<GROUP>, D = 8 / UNIT;
    extern __shared__ __align__(128) uint8_t rows_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kbs = w.blocks(), groups = w.groups(), units = kbs / UNIT, row_bytes = w4r_row_bytes(kbs), row_tiles = w.row_tiles();
    uint32_t* tops = reinterpret_cast<uint32_t*>(rows_smem + 16);
    uint8_t* batch = rows_smem + W4R_HEAD;
    float* sums = reinterpret_cast<float*>(batch + 8 * row_bytes);
    const uint32_t bar = smem_addr(rows_smem);
    if (threadIdx.x == 0) {
        mbar_init(bar, 1);
        fence_barrier_init();
        fence_proxy_async();
    }
    if (threadIdx.x < 16) tops[threadIdx.x] = 0;
    if (w.k & 63 && threadIdx.x < 32)              // the rest of a row's last block
        *reinterpret_cast<uint4*>(batch + (threadIdx.x >> 2) * row_bytes + w.k * 2 + (threadIdx.x & 3) * 16) = make_uint4(0u, 0u, 0u, 0u);
    pdl_trigger();
    pdl_wait();
    const int count = tiles.count();
    int total = 0;                                 // items
    for (int i0 = 0; i0 < count; i0 += 32) {
        const int i = i0 + lane;
        total += __reduce_add_sync(0xffffffffu, i < count ? (tiles.at(i).rows + 7) >> 3 : 0);
    }
    // As many shares of K as leave a CTA W4E_STEPS steps or fewer (4 of 32 experts of 5760 x 2880, 4 tokens: 3 steps 27, 6 29, 12 32 us).
    int wk_shift = 3;
    while (wk_shift > 0 && ((long)total * row_tiles >> (3 - wk_shift) > (long)W4E_STEPS * gridDim.x || units >> wk_shift == 0)) --wk_shift;
    const int wr_shift = 3 - wk_shift, wk = 1 << wk_shift, share = warp & (wk - 1);
    const int per_item = (row_tiles + (1 << wr_shift) - 1) >> wr_shift;            // steps
    const long all = (long)total * per_item;
    const long begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
    if (begin >= end) return;

    // Where a step is: entry of the list, chunk of its rows, row tiles.
    struct Place {
        int entry, chunk, at;
        W4Item item;
    } there{0, 0, (int)(begin % per_item), W4Item{0, 0, 0}};
    int skip = (int)(begin / per_item);
    for (int i0 = 0;; i0 += 32) {                  // (ends: begin is less than the items' steps)
        const int i = i0 + lane, mine = i < count ? (tiles.at(i).rows + 7) >> 3 : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, upto > skip);
        if (past) {
            const int l = __ffs(past) - 1;
            there.entry = i0 + l;
            there.chunk = skip - __shfl_sync(0xffffffffu, upto - mine, l);
            break;
        }
        skip -= __shfl_sync(0xffffffffu, upto, 31);
        if (i0 + 32 >= count) return;
    }
    there.item = tiles.at(there.entry);
    auto next = [&](Place& p) {                    // whether that is another item
        if (++p.at < per_item) return false;
        p.at = 0;
        if (++p.chunk * 8 >= p.item.rows) {
            p.chunk = 0;
            do p.item = ++p.entry < count ? tiles.at(p.entry) : W4Item{0, 1, 0};
            while (p.item.rows == 0);
        }
        return true;
    };

    // Codes on their way: D units per lane; the next step's first are asked for before this one's sums meet.
    const int mine = (units - share + wk - 1) >> wk_shift;        // units of this warp in a step
    Place here = there;                            // where the sums are; `there` is where the fetches are
    uint4 c[D][UNIT];
    uint32_t s[D][SETS];
    uint16_t z[D][SETS];
    const uint4* codes = nullptr;
    const uint32_t* scale = nullptr;
    const uint16_t* zero = nullptr;
    const int code_step = wk * UNIT * 256, set_step = wk * SETS * 64, x_step = wk * UNIT * 128;
    int steps = (int)(end - begin);
    auto fetch = [&](int d) {
#pragma unroll
        for (int v = 0; v < UNIT; ++v) c[d][v] = ld_stream(codes + v * 256);
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            s[d][u] = __ldg(scale + u * 64);
            if (KIND == W4_ZERO) z[d][u] = __ldg(zero + u * 64);
        }
        codes += code_step;
        scale += set_step;
        zero += set_step;
    };
    auto aim = [&]() {                             // at a step's codes, and the first of them
        const int rt = min((there.at << wr_shift) + (warp >> wk_shift), w.panels() * 8 - 1);
        const size_t panel = (size_t)there.item.expert * w.panels() + (rt >> 3);
        const size_t set = ((panel * groups + share * SETS) * 8 + (rt & 7)) * 8 + g;
        codes = w.codes + ((panel * kbs + share * UNIT) * 8 + (rt & 7)) * 32 + lane;
        scale = w.scale + set;
        zero = w.zero + set;
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < mine) fetch(d);
    };
    aim();

    // thread's four features of a step's, and its row
    const int r4 = (threadIdx.x & ((4 << wr_shift) - 1)) * 4, col = threadIdx.x >> (2 + wr_shift);
    bool ok = true;
    uint32_t parity = 0, *top = tops;
    const uint8_t* x0 = batch;
    int rows = 0, row0 = 0;
    float4 f;
    float acc[1][4];
    const uint8_t* xr[1];
    auto enter = [&](bool fresh) {                 // a step
        if (fresh) {                               // the item's rows; everyone is done with the last one's
            rows = min(8, here.item.rows - here.chunk * 8);
            row0 = here.item.row0 + here.chunk * 8;
            if (warp == 0) {
                if (lane == 0) {
                    fence_proxy_async();           // the copies write where the threads have written
                    mbar_arrive_expect_tx(bar, rows * w.k * 2);
                }
                __syncwarp();
                if (lane < rows) bulk_load(smem_addr(batch) + lane * row_bytes, x + (size_t)(row0 + lane) * ldx, w.k * 2, bar);
            }
            if (!mbar_wait(bar, parity, status, PIE_ERR_WAIT_TMA)) {
                drain(bar, parity);
                ok = false;
            }
            if (KIND == W4_FP4) {
                top = tops + parity * 8;           // everyone was done with the other ones before the last step's barrier
                w4_batch_fp16(batch, row_bytes, rows, w.k >> 3, top);
                if (threadIdx.x < 8) tops[(parity ^ 1u) * 8 + threadIdx.x] = 0;
            }
            parity ^= 1u;
            x0 = batch + min(g, rows - 1) * row_bytes + share * UNIT * 128 + t * 16;
        }
        const int f0 = (here.at << (wr_shift + 4)) + r4;
        f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (col < rows && f0 < w.n) f = __ldg(reinterpret_cast<const float4*>(w.factor + (size_t)here.item.expert * w.panels() * 128 + f0));
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][j] = 0.f;
        xr[0] = x0;
        __syncwarp();                              // lanes leave the wait and the last step's stores one by one; an MMA is all of theirs
    };
    auto leave = [&]() {                           // false where a wait ran out
        if (KIND == W4_FP4) w4_unscale(acc[0], top + 2 * t);
        float* part = sums + (steps & 1) * 64 * W4R_PAD;
        float* mine_at = part + (warp * 8 + 2 * t) * W4R_PAD + g;
        mine_at[0] = acc[0][0];
        mine_at[W4R_PAD] = acc[0][1];
        mine_at[8] = acc[0][2];
        mine_at[W4R_PAD + 8] = acc[0][3];
        if (!__syncthreads_and(ok)) return false;
        const int f0 = (here.at << (wr_shift + 4)) + r4;
        if (col < rows && f0 < w.n) {
            const float* from = part + (((r4 >> 4) << wk_shift) * 8 + col) * W4R_PAD + (r4 & 15);
            float4 v = *reinterpret_cast<const float4*>(from);
            for (int k = 1; k < wk; ++k) {
                const float4 y = *reinterpret_cast<const float4*>(from + k * 8 * W4R_PAD);
                v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
            }
            v.x *= f.x * W4_UNIT<KIND>; v.y *= f.y * W4_UNIT<KIND>; v.z *= f.z * W4_UNIT<KIND>; v.w *= f.w * W4_UNIT<KIND>;
            bf16* to = C + (size_t)(row0 + col) * ldc;
            if (epi == EPI_SWIGLU) {
                const float a = glu_value<EPI_SWIGLU>(v.x, v.y, 0.f), b = glu_value<EPI_SWIGLU>(v.z, v.w, 0.f);
                *reinterpret_cast<bf162*>(to + (f0 >> 1)) = __floats2bfloat162_rn(a, b);
            } else {
                const bf162 o[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
                *reinterpret_cast<uint2*>(to + f0) = *reinterpret_cast<const uint2*>(o);
            }
        }
        return true;
    };
    __syncthreads();
    for (bool fresh = true; steps > 0; --steps, fresh = next(here)) {
        enter(fresh);
        for (int left = mine; left > 0; left -= D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (d >= left) break;
                w4_unit<KIND, GROUP, 1>(c[d], s[d], z[d], xr, acc);
                xr[0] += x_step;
                if (D + d < left) fetch(d);
            }
        }
        if (steps > 1) {
            next(there);
            aim();
        }
        if (!leave()) return;
    }
}

// ------------------------------------------------------------------ more rows
// tcgen05: 128 weight rows are the MMA's rows and come from tensor memory, where eight warps put them expanded to fp16, straight from
// registers; up to 128 rows of the batch are its columns, brought by TMA. Shared memory so holds the weights' codes only, and a weight is
// expanded once per 128 rows of the batch (256 leave an SM one CTA: no faster for one weight, 5 to 30 % slower over experts).
//
// Why fp16: an integer of -8 .. 7 times a bf16 scale fits its 11 bits, others (zero points, fp16 scales) are off by 2^-11 of the weight at most,
// where bf16 operands would round each weight by 2^-8. The batch's rows go there by w4_rows_fp16_kernel, each times a power of two that brings
// its largest value to [2^14, 2^15): a bf16 value keeps all its bits down to 2^-29 of the row's largest.
//
// K is split over the CTAs of a cluster where there are few tiles, as in gemm_skinny.cu; partial tiles meet in distributed shared memory
// in CTA order. Every mbarrier wait is bounded.
//
// Bound by the MMA issuer's way through two blocks: 690 cycles at 48 columns (clocks read in the kernel: its two waits 185 although what they
// wait for is there, eight MMAs 230, two commits and the loop the rest), 900 at 128, where the MMAs themselves are 192 and 512 by the rate and
// the expansion of their weights 600; two CTAs of an SM hide a part of that from each other. 2048 rows through 28672 x 4096: 391 us in a
// graph, 74 % of the rate of a library product of bf16 measured in bursts (calls one after another run into the power limit: 459 us); 48 rows through
// 6144 x 4096 11.4 us with the conversion, 4096 x 14336 19, 28672 x 4096 23.
using namespace sm100;

// Work of a launch, in items of up to tile_rows rows: rows [0, M) of one weight, or the rows of a sorted batch (tiles as in gemm_grouped.cu),
// whose items w4_rows_fp16_kernel lists: [0] their number, then (first row, rows, expert) each.
struct W4Work {
    int4* items;                              // null: one weight
    int M, tile_rows;
};
__device__ __forceinline__ int w4_items(const W4Work& w) { return w.items ? w.items[0].x : (w.M + w.tile_rows - 1) / w.tile_rows; }
__device__ __forceinline__ W4Item w4_item(const W4Work& w, int i) {
    if (w.items) {
        const int4 v = w.items[1 + i];
        return W4Item{v.x, v.y, v.z};
    }
    return W4Item{i * w.tile_rows, min(w.tile_rows, w.M - i * w.tile_rows), 0};
}

// A block per row: out = fp16(x 2^e), back[row] = 2^-e. Infinities and NaN stay what they are and do not count for e. Columns go where the
// codes' layout has them: of 32 columns, 8 t + 4 h .. + 3 to 16 h + 4 t. The row stays in registers (up to VECS * 2048 columns; longer
// ones are read again).
template <int VECS>
__global__ void __launch_bounds__(256) w4_rows_fp16_kernel(const bf16* x, int ldx, __half* __restrict__ out, float* __restrict__ back,
                                                           int K, int pitch, const W4Work work, const W4Tiles tiles) {
    __shared__ float red[8];
    pdl_trigger();
    pdl_wait();
    W4Item t{0, work.M, 0};
    if (work.items) {
        const int count = tiles.count();
        if (blockIdx.x == gridDim.x - 1) {             // a block of its own lists the items, a warp of it
            if (blockIdx.y != 0 || threadIdx.x >= 32) return;
            int total = 0;
            for (int i0 = 0; i0 < count; i0 += 32) {
                const int i = i0 + (int)threadIdx.x;
                const W4Item e = i < count ? tiles.at(i) : W4Item{0, 0, 0};
                const int mine = (e.rows + work.tile_rows - 1) / work.tile_rows;
                int before = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, before, o);
                    if ((int)threadIdx.x >= o) before += v;
                }
                for (int j = 0, at = 0; j < mine; ++j, at += work.tile_rows)
                    work.items[1 + total + before - mine + j] = make_int4(e.row0 + at, min(work.tile_rows, e.rows - at), e.expert, 0);
                total += __shfl_sync(0xffffffffu, before, 31);
            }
            if (threadIdx.x == 0) work.items[0] = make_int4(total, 0, 0, 0);
            return;
        }
        if ((int)blockIdx.x >= count) return;
        t = tiles.at(blockIdx.x);
    }
    const int vecs = K >> 3;                                   // K is a multiple of 32
    for (int r = blockIdx.y; r < t.rows; r += gridDim.y) {
        const size_t row = (size_t)(t.row0 + r);
        const bf16x8* src = reinterpret_cast<const bf16x8*>(x + row * ldx);
        bf16x8 v[VECS];
        float amax = 0.f;
        auto peak = [&](const bf16x8& p) {
            float f[8];
            unpack8(p, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.f);
        };
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int at = threadIdx.x + i * 256;
            if (at < vecs) v[i] = src[at];
        }
#pragma unroll
        for (int i = 0; i < VECS; ++i)
            if ((int)threadIdx.x + i * 256 < vecs) peak(v[i]);
        for (int at = threadIdx.x + VECS * 256; at < vecs; at += 256) peak(src[at]);
        amax = warp_max(amax);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
        __syncthreads();
        amax = red[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) amax = fmaxf(amax, red[i]);
        __syncthreads();
        const int top = (int)(__float_as_uint(amax) >> 23) - 127;          // exponent of the largest (-127 for zero and subnormals)
        const int e = amax > 0.f ? max(-126, min(126, 14 - top)) : 0;
        const float f = exp2_int(e);
        __half* dst = out + row * pitch;                                    // padded with zeros to 64 columns
        if (pitch > K && threadIdx.x < 4) *reinterpret_cast<uint4*>(dst + K + threadIdx.x * 8) = make_uint4(0u, 0u, 0u, 0u);
        auto store = [&](const bf16x8& p, int at) {
            float y[8];
            unpack8(p, y);
            __half2 h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(y[2 * j] * f, y[2 * j + 1] * f);
            __half* to = dst + (at >> 2) * 32 + (at & 3) * 4;
            *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(h);
            *reinterpret_cast<uint2*>(to + 16) = *reinterpret_cast<const uint2*>(h + 2);
        };
#pragma unroll
        for (int i = 0; i < VECS; ++i)
            if ((int)threadIdx.x + i * 256 < vecs) store(v[i], threadIdx.x + i * 256);
        for (int at = threadIdx.x + VECS * 256; at < vecs; at += 256) store(src[at], at);
        if (threadIdx.x == 0) back[row] = exp2_int(-e);
    }
}

// The scale of a row and group as the expansion wants it, and a pair of weights in fp16, times W4_HALF_UNIT<KIND>. As in w4_pair the bits of a
// code are the subnormal number q 2^-24, or q 2^-20 four bits higher.
//   W4_INT   q 2^-24 * s + (-8 s 2^-24): one rounding, of the result, as the addend is exact. Scales of a row are within 2^5 of each
//            other (others come with zero points of 8), so the result has 9 bits or more.
//   W4_ZERO  (q - z) / 2^9 exactly, times s
//   W4_FP4   the number, times s
template <int KIND>
constexpr float W4_HALF_UNIT = KIND == W4_INT ? 16777216.f : KIND == W4_ZERO ? 512.f : 1.f;
template <int KIND>
struct W4Half {
    __half2 lo, hi, zero;
    // s: the row's scale, twice; z: zero points, of which byte i
    __device__ __forceinline__ W4Half(__half2 s, uint32_t z, int i) {
        if (KIND == W4_INT) {
            lo = s;
            hi = __hmul2(s, half2_bits(0x2c002c00u));                       // 2^-4
            zero = __hmul2(__hmul2(s, half2_bits(0x04000400u)), half2_bits(0xa000a000u));       // -2^-21, in two steps that are exact
        } else {
            lo = hi = s;
            if (KIND == W4_ZERO) zero = __hmul2(half2_bits(__byte_perm(z, 0u, i ? 0x4141 : 0x4040)), half2_bits(0xf800f800u));        // -z 2^-9
        }
    }
    __device__ __forceinline__ uint32_t pair(uint32_t word, int i) const {          // of e2m1, word is the pair in fp16
        __half2 r;
        if (KIND == W4_FP4) {
            r = __hmul2(half2_bits(word), lo);
        } else {
            const __half2 v = half2_bits((i < 2 ? word : word >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu));
            if (KIND == W4_INT) r = __hfma2(v, i & 1 ? hi : lo, zero);
            else r = __hmul2(__hfma2(v, half2_bits(i & 1 ? 0x68006800u : 0x78007800u), zero), lo);
        }
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

// A in tensor memory (fp16 pairs, one 32-bit column each), B in shared memory.
__device__ __forceinline__ void umma_f16_tmem_a(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 lanes x 32 columns: four blocks of eight columns, in each of which lane 4 g + t has columns 2 t, 2 t + 1 of TMEM lanes g (v[0], v[1])
// and g + 8 (v[2], v[3]).
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

constexpr int W4T_THREADS = 320;
constexpr int W4T_A_STAGES = 3;                                    // most stages of weights, two blocks each
constexpr int W4T_X_STAGES = 8, W4T_C_STAGES = 4;                  // most stages of the batch and of codes
constexpr int W4T_CHUNK = 4;                                       // blocks of 64 columns per stage of codes
constexpr uint32_t W4T_A_COLS = GEMM_BK / 2;                       // TMEM columns of a block of weights
constexpr uint32_t W4T_BAR_BYTES = 256;
// A stage of codes: 128 rows' codes, scales and zero points.
template <int KIND, int GROUP>
constexpr uint32_t W4T_C_BYTES = 8 * (W4T_CHUNK * 512 + W4T_CHUNK * 64 / GROUP * (KIND == W4_ZERO ? 48 : 32));
// The batch's stages and the partial tiles of a cluster share memory: what the latter need.
__host__ __device__ constexpr uint32_t w4_join_bytes(int cols) { return 512u * (uint32_t)cols + 8192u; }

__device__ __forceinline__ bool all_of_warp(bool yes) { return __all_sync(0xffffffffu, yes); }

// The batch's rows as [blocks of 64 columns][rows][64 columns], in boxes of a stage's blocks and, of a sorted batch, 16, 32, 64 or 128
// rows; else the first map has the rows of an item.
struct W4Maps {
    CUtensorMap x[4];
};
__device__ __forceinline__ int w4_box(const W4Work& w, const W4Item& t) { return w.items && t.rows > 16 ? 28 - __clz(t.rows - 1) : 0; }
__device__ __forceinline__ uint32_t w4_box_rows(const W4Work& w, int box) { return w.items ? 16u << box : (uint32_t)w.tile_rows; }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void w4_store(int epi, const float (&v)[16], int feat, int tok0, int F, int tok_end, bf16* C, int ldc,
                                         const bf16* R, int ldr) {
    const EpiArgs ex;
    const XieluCoef act(nullptr);
    if (epi == EPI_SWIGLU) skinny_store<EPI_SWIGLU>(v, feat, tok0, F, tok_end, C, ldc, R, ldr, ex, act);
    else if (epi == EPI_GEGLU) skinny_store<EPI_GEGLU>(v, feat, tok0, F, tok_end, C, ldc, R, ldr, ex, act);
    else if (epi == EPI_RESIDUAL) skinny_store<EPI_RESIDUAL>(v, feat, tok0, F, tok_end, C, ldc, R, ldr, ex, act);
    else skinny_store<EPI_STORE>(v, feat, tok0, F, tok_end, C, ldc, R, ldr, ex, act);
}

// Shape of a launch: most columns of an item, CTAs that share an item's K, stages.
struct W4Shape {
    int room, splits, x_blocks, x_stages, c_stages;        // x_blocks: blocks of 64 columns per stage of the batch (1, 2 or 4)
};

// Roles: warp 0 loads the batch and the codes, warp 1 issues MMAs, warps 2-9 expand codes and store results.
template <int KIND, int GROUP>
__global__ void __launch_bounds__(W4T_THREADS, 2)
w4_tile_kernel(const __grid_constant__ W4Maps maps, const W4Weight w, const float* back, bf16* C, int ldc, const bf16* R, int ldr, const W4Work work,
               const W4Shape shape, int epi, int* status) {
    constexpr int UNIT = GROUP == 128 ? 2 : 1;                      // a CTA's share of K has whole groups
    constexpr uint32_t SETS = W4T_CHUNK * 64 / GROUP, SCALE_AT = 8 * W4T_CHUNK * 512, ZERO_AT = SCALE_AT + 8 * SETS * 32;
    constexpr uint32_t C_BYTES = W4T_C_BYTES<KIND, GROUP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t* ring_ptr = smem_raw + (ring - raw);
    const int room = shape.room, splits = shape.splits, xb = shape.x_blocks, xs = shape.x_stages, cs = shape.c_stages;
    const uint32_t x_bytes = (uint32_t)room * (GEMM_BK * 2), x_stage = x_bytes * xb;
    const uint32_t x_total = max(xs * x_stage, splits > 1 ? w4_join_bytes(room) : 0u);
    const uint32_t code_ring = ring + x_total;
    const uint8_t* code_ptr = ring_ptr + x_total;
    const uint32_t bar0 = code_ring + cs * C_BYTES;
    auto xfull = [&](int s) { return bar0 + 8u * s; };
    auto xempty = [&](int s) { return bar0 + 8u * (W4T_X_STAGES + s); };
    auto cfull = [&](int s) { return bar0 + 8u * (2 * W4T_X_STAGES + s); };
    auto cempty = [&](int s) { return bar0 + 8u * (2 * W4T_X_STAGES + W4T_C_STAGES + s); };
    auto afull = [&](int s) { return bar0 + 8u * (2 * W4T_X_STAGES + 2 * W4T_C_STAGES + s); };
    auto aempty = [&](int s) { return bar0 + 8u * (2 * W4T_X_STAGES + 2 * W4T_C_STAGES + W4T_A_STAGES + s); };
    constexpr int BARS = 2 * (W4T_X_STAGES + W4T_C_STAGES + W4T_A_STAGES);
    static_assert((BARS + 2) * 8 + 4 <= W4T_BAR_BYTES + 64, "barriers");
    const uint32_t dfull = bar0 + 8u * BARS, dempty = dfull + 8u;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ring_ptr + x_total + cs * C_BYTES + 8 * (BARS + 2));

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const uint32_t d_cols = room <= 64 ? 64u : 128u, a_stages = room <= 64 ? 3u : 2u;
    constexpr uint32_t tmem_cols = 256;
    const int tiles_n = w.panels(), kbs = w.blocks(), groups = w.groups();
    const int part = splits > 1 ? (int)cluster_ctarank() : 0, units = kbs / UNIT;
    const int kb0 = (int)((long)units * part / splits) * UNIT, nb = (int)((long)units * (part + 1) / splits) * UNIT - kb0;
    const int first_item = blockIdx.x / splits, item_step = gridDim.x / splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < xs; ++s) {
            mbar_init(xfull(s), 1);
            mbar_init(xempty(s), 1);
        }
        for (int s = 0; s < cs; ++s) {
            mbar_init(cfull(s), 1);
            mbar_init(cempty(s), 8);
        }
        for (int s = 0; s < W4T_A_STAGES; ++s) {
            mbar_init(afull(s), 4);
            mbar_init(aempty(s), 1);
        }
        mbar_init(dfull, 1);
        mbar_init(dempty, 8);
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) {
        tmem_alloc(smem_addr(const_cast<uint32_t*>(tmem_slot)), tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // (the shuffle tells the compiler that it is uniform: MMA operands that are not are moved to uniform registers one by one)
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0), a_base = tmem_base + d_cols;
    pdl_trigger();
    if (work.items) pdl_wait();                    // the list is a launch's ahead; a weight is not
    const int items = w4_items(work) * tiles_n;

    if (warp == 0) {
        if (elect_one()) {
            // The codes' stages run `cs` ahead of the batch's, which wait for the MMAs: a stage of codes is free when it has been expanded,
            // which is before its MMAs are done.
            bool ok = true;
            uint32_t cit = 0, c = 0, cph = 0;
            int c_item = first_item, c_at = 0;
            W4Item ct{0, 0, 0};
            auto codes = [&]() {
                if (c_item >= items || nb == 0) return;
                if (c_at == 0) ct = w4_item(work, c_item / tiles_n);
                if (!mbar_wait(cempty(c), cph ^ 1u, status, PIE_ERR_WAIT_TMA)) { ok = false; return; }
                const int blocks = min(W4T_CHUNK, nb - c_at), sets = blocks * 64 / GROUP, kb = kb0 + c_at;
                const size_t panel = (size_t)ct.expert * tiles_n + c_item % tiles_n, set = (panel * groups + kb * 64 / GROUP) * 8;
                mbar_arrive_expect_tx(cfull(c), 8u * (blocks * 512 + sets * (KIND == W4_ZERO ? 48 : 32)));
                const uint32_t dst = code_ring + c * C_BYTES;
                bulk_load(dst, w.codes + (panel * kbs + kb) * 256, blocks * 4096, cfull(c));
                bulk_load(dst + SCALE_AT, w.scale + set * 8, sets * 256, cfull(c));
                if (KIND == W4_ZERO) bulk_load(dst + ZERO_AT, w.zero + set * 8, sets * 128, cfull(c));
                ++cit;
                if (++c == (uint32_t)cs) { c = 0; cph ^= 1u; }
                c_at += W4T_CHUNK;
                if (c_at >= nb) { c_at = 0; c_item += item_step; }
            };
            for (int i = 0; i < cs; ++i) codes();
            pdl_wait();
            uint32_t it = 0, s = 0, ph = 0;
            for (int item = first_item; item < items && ok; item += item_step) {
                const W4Item t = w4_item(work, item / tiles_n);
                const int box = w4_box(work, t);
                const uint32_t rows = w4_box_rows(work, box);
                for (int at = 0; at < nb && ok; at += xb, ++it) {
                    if (!mbar_wait(xempty(s), ph ^ 1u, status, PIE_ERR_WAIT_TMA)) { ok = false; break; }
                    mbar_arrive_expect_tx(xfull(s), rows * xb * (GEMM_BK * 2));        // blocks past the last and rows past the batch's are filled in
                    tma_load_3d(ring + s * x_stage, &maps.x[box], xfull(s), 0, t.row0, kb0 + at);
                    if (++s == (uint32_t)xs) { s = 0; ph ^= 1u; }
                    if ((at & (W4T_CHUNK - 1)) + xb == W4T_CHUNK || at + xb >= nb) codes();      // one stage of codes per stage's worth of the batch
                }
            }
            // no copy may be in flight when a ring is reused or the CTA exits
            const uint32_t first = it > (uint32_t)xs ? it - xs : 0u, c_first = cit > (uint32_t)cs ? cit - cs : 0u;
            for (uint32_t j = first; j < it; ++j) drain(xfull(j % xs), (j / xs) & 1u);
            for (uint32_t j = c_first; j < cit; ++j) drain(cfull(j % cs), (j / cs) & 1u);
        }
    } else if (warp == 1) {
        {
            // the whole warp walks the loop, so that it is uniform to the compiler; one lane issues
            const bool leader = elect_one();
            uint32_t count = 0, s = 0, ph = 0, as = 0, aph = 0;
            bool ok = true;
            for (int item = first_item; item < items && ok; item += item_step) {
                const W4Item t = w4_item(work, item / tiles_n);
                // fp16 x fp16 -> fp32: both operand formats 0
                const uint32_t idesc = (1u << 4) | ((uint32_t)((t.rows + 15) / 16 * 2) << 17) | ((uint32_t)(GEMM_BM >> 4) << 24);
                const uint32_t x_block = w4_box_rows(work, w4_box(work, t)) * (GEMM_BK * 2);
                if (!all_of_warp(mbar_wait(dempty, (count & 1u) ^ 1u, status, PIE_ERR_WAIT_EPILOGUE))) break;
                ++count;
                tc_fence_after();
                // Two blocks at a time, as the weights come; both halves of a stage of codes, also where the second has no block: its stage
                // changes hands all the same.
                for (int at = 0; at < (nb + W4T_CHUNK - 1) / W4T_CHUNK * W4T_CHUNK; at += 2) {
                    if (at < nb && !all_of_warp(mbar_wait(xfull(s), ph, status, PIE_ERR_WAIT_TMA))) { ok = false; break; }
                    if (!all_of_warp(mbar_wait(afull(as), aph, status, PIE_ERR_WAIT_TMA))) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a = a_base + as * (2 * W4T_A_COLS);
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        if (at + d >= nb) break;
                        if (d == 1 && xb == 1) {
                            if (!all_of_warp(mbar_wait(xfull(s), ph, status, PIE_ERR_WAIT_TMA))) { ok = false; break; }
                            tc_fence_after();
                        }
                        const uint64_t xd = make_smem_desc_sw128(ring + s * x_stage + (xb == 2 ? d * x_block : 0u));
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < GEMM_BK / 16; ++k)
                                umma_f16_tmem_a(tmem_base, a + d * W4T_A_COLS + 8 * k, xd + 2u * k, idesc, (at | d | k) != 0);
                        }
                        if (d == 1 || xb == 1 || at + 1 >= nb) {
                            if (leader) umma_commit(xempty(s));
                            if (++s == (uint32_t)xs) { s = 0; ph ^= 1u; }
                        }
                    }
                    if (!ok) break;
                    if (leader) umma_commit(aempty(as));
                    if (++as == a_stages) { as = 0; aph ^= 1u; }
                }
                if (ok && leader) umma_commit(dfull);
                __syncwarp();
            }
        }
    } else {
        // Warps 2-5 expand the first two blocks of a stage of codes, warps 6-9 the others; a warp its two row tiles (TMEM lanes 32 q ..).
        const int q = warp & 3, odd = (warp - 2) >> 2, g8 = lane >> 2;
        uint32_t count = 0, s = 0, ph = 0;                  // items, stage of codes
        uint32_t as = (uint32_t)odd, aph = 0;               // stage of weights: every second one is this half's
        bool ok = true;
        for (int item = first_item; item < items && ok; item += item_step) {
            const W4Item t = w4_item(work, item / tiles_n);
            const int tile_n = item % tiles_n;
            // a wait that ran out makes the later ones end soon; what they leave is wrong and not stored
            for (int at = 0; at < nb; at += W4T_CHUNK) {
                ok &= mbar_wait(cfull(s), ph, status, PIE_ERR_WAIT_TMA);
                const uint8_t* stage = code_ptr + s * C_BYTES;
                const uint32_t dst = a_base + as * (2 * W4T_A_COLS) + ((uint32_t)(q * 32) << 16);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = 2 * odd + i;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 c = *reinterpret_cast<const uint4*>(stage + d * 4096 + (q * 2 + h) * 512 + lane * 16);
                        const uint32_t word[4] = {c.x, c.y, c.z, c.w};
                        uint32_t o[16];
#pragma unroll
                        for (int u = 0; u < (GROUP == 32 ? 2 : 1); ++u) {
                            const int set = GROUP == 128 ? odd : GROUP == 64 ? d : 2 * d + u;
                            const __half2 f = *reinterpret_cast<const __half2*>(stage + SCALE_AT + set * 256 + (q * 2 + h) * 32 + g8 * 4);
                            uint32_t z = 0u;
                            if (KIND == W4_ZERO) z = *reinterpret_cast<const uint16_t*>(stage + ZERO_AT + set * 128 + (q * 2 + h) * 16 + g8 * 2);
                            const W4Half<KIND> r0(__low2half2(f), z, 0), r1(__high2half2(f), z, 1);
#pragma unroll
                            for (int j = (GROUP == 32 ? 2 * u : 0); j < (GROUP == 32 ? 2 * u + 2 : 4); ++j) {
                                uint32_t v[4] = {word[j], word[j], word[j], word[j]};
                                if (KIND == W4_FP4) e2m1_pairs(word[j], v);
                                o[4 * j] = r0.pair(v[0], 0);
                                o[4 * j + 1] = r0.pair(v[1], 1);
                                o[4 * j + 2] = r1.pair(v[2], 2);
                                o[4 * j + 3] = r1.pair(v[3], 3);
                            }
                        }
                        if (i == 0 && h == 0) {              // the MMAs are done with what both blocks replace
                            ok &= mbar_wait(aempty(as), aph ^ 1u, status, PIE_ERR_WAIT_MMA);
                            tc_fence_after();
                            __syncwarp();
                        }
                        // (a block past the last is expanded from what the ring holds and not multiplied)
                        tmem_st_16x256b_x4(dst + i * W4T_A_COLS + (h ? 16u << 16 : 0u), o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(afull(as));
                    mbar_arrive(cempty(s));
                }
                as += 2;
                if (as >= a_stages) { as -= a_stages; aph ^= 1u; }
                if (++s == (uint32_t)cs) { s = 0; ph ^= 1u; }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (splits > 1) break;           // one item per cluster; the tile is joined below
            pdl_wait();                      // outputs, residual and row factors may still be in use
            const bool got = ok && mbar_wait(dfull, count & 1u, status, PIE_ERR_WAIT_MMA);
            ++count;
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after();
            const int feat = tile_n * GEMM_BM + q * 32 + lane;
            const float rf = feat < w.n ? w.factor[(size_t)t.expert * tiles_n * GEMM_BM + feat] * W4_HALF_UNIT<KIND> : 0.f;
            const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16);
            for (int g = odd; g * 16 < t.rows; g += 2) {
                uint32_t r[16];
                float v[16];
                __syncwarp();                // features past the last store nothing
                tmem_ld_32x16(t_row + g * 16, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) * (rf * back[t.row0 + min(g * 16 + j, t.rows - 1)]);
                w4_store(epi, v, feat, g * 16, w.n, t.rows, C + (size_t)t.row0 * ldc, ldc, R + (size_t)t.row0 * ldr, ldr);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dempty);
        }
    }
    if (splits > 1) {
        // Units of 32 features x 16 tokens; unit u is summed and stored by CTA u % splits, from partials that lie in its ring as
        // [unit / splits][source][4 tokens][32 features].
        const W4Item t = w4_item(work, first_item / tiles_n);
        const int q = warp & 3, odd = (warp - 2) >> 2, chunks = (t.rows + 15) / 16, tile_n = first_item % tiles_n;
        const bool worker = warp >= 2;
        bool got = true;
        if (worker) {
            got = __all_sync(0xffffffffu, mbar_wait(dfull, 0, status, PIE_ERR_WAIT_MMA));
            tc_fence_after();
        }
        __syncwarp();
        cluster_sync_all();              // every ring of the cluster is free, and every CTA has started
        if (worker && got) {
            for (int g = odd; g < chunks; g += 2) {
                uint32_t r[16];
                tmem_ld_32x16(tmem_base + ((uint32_t)(q * 32) << 16) + g * 16, r);
                tmem_ld_wait();
                const int u = q * chunks + g;
                const uint32_t at = map_to_cta(ring + (uint32_t)((u / splits * splits + part) * 2048 + lane * 16), (uint32_t)(u % splits));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    st_cluster_v4(at + j * 512, __uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                  __uint_as_float(r[4 * j + 3]));
            }
        }
        tc_fence_before();
        __syncwarp();
        cluster_sync_all();
        if (worker && got) {
            pdl_wait();
            for (int slot = warp - 2; slot * splits + part < 4 * chunks; slot += 8) {
                const int u = slot * splits + part, feat = tile_n * GEMM_BM + u / chunks * 32 + lane, g = u % chunks;
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
                for (int src = 0; src < splits; ++src) {
                    const float4* p = reinterpret_cast<const float4*>(ring_ptr + (slot * splits + src) * 2048) + lane;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 a = p[j * 32];
                        v[4 * j] += a.x; v[4 * j + 1] += a.y; v[4 * j + 2] += a.z; v[4 * j + 3] += a.w;
                    }
                }
                const float rf = feat < w.n ? w.factor[(size_t)t.expert * tiles_n * GEMM_BM + feat] * W4_HALF_UNIT<KIND> : 0.f;
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] *= rf * back[t.row0 + min(g * 16 + j, t.rows - 1)];
                w4_store(epi, v, feat, g * 16, w.n, t.rows, C + (size_t)t.row0 * ldc, ldc, R + (size_t)t.row0 * ldr, ldr);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

}  // namespace pie

using namespace pie;

// Lets a kernel have all of an SM's shared memory, once per device.
template <typename Kernel>
static cudaError_t w4_all_smem(Kernel kern, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) & bit))) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// A product's operands beside the weight.
struct W4Call {
    const bf16* x;
    int ldx;
    bf16* C;
    int ldc;
    const bf16* R;
    int ldr, M, epi;
    int *status, num_sms;
    cudaStream_t st;
};

static int w4_check(const W4Weight& w) {
    const bool group = w.group == 32 || w.group == 64 || w.group == 128;
    return w.experts < 0 || w.n <= 0 || w.k <= 0 || !group || w.k % w.group ? (int)cudaErrorInvalidValue : 0;
}
// Rows on 16-byte boundaries, N a multiple of 8 (32 behind a GLU).
static int w4_check(const W4Weight& w, const W4Call& c) {
    if (int e = w4_check(w)) return e;
    const bool glu = c.epi == EPI_SWIGLU || c.epi == EPI_GEGLU;
    if (!glu && c.epi != EPI_STORE && c.epi != EPI_RESIDUAL) return (int)cudaErrorInvalidValue;
    if (c.ldx % 8 || c.ldc % 8 || w.n % (glu ? 32 : 8)) return (int)cudaErrorInvalidValue;
    return c.epi == EPI_RESIDUAL && (!c.R || c.ldr % 8) ? (int)cudaErrorInvalidValue : 0;
}
// A launch under programmatic dependence, of clusters of `ctas`.
template <typename... KArgs, typename... Args>
static cudaError_t w4_launch(void (*kern)(KArgs...), dim3 grid, int threads, int smem, int ctas, cudaStream_t st, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_pie_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// The weight (all experts of it) in bf16, row-major [experts][n][k].
PIE_API int pie_w4_expand(const void* weight, void* out, cudaStream_t st) {
    const W4Weight& w = *reinterpret_cast<const W4Weight*>(weight);
    if (int e = w4_check(w)) return e;
    if (w.experts == 0) return 0;
    const long tiles = (long)w.experts * w.panels() * w.blocks() * 8;
    const int blocks = (int)min((tiles + 7) / 8, (long)PIE_SMS * 8);
    switch (w4_kind(w)) {
        case W4_FP4: w4_expand_kernel<W4_FP4><<<blocks, 256, 0, st>>>(w, (bf16*)out); break;
        case W4_ZERO: w4_expand_kernel<W4_ZERO><<<blocks, 256, 0, st>>>(w, (bf16*)out); break;
        default: w4_expand_kernel<W4_INT><<<blocks, 256, 0, st>>>(w, (bf16*)out);
    }
    return (int)cudaGetLastError();
}

// CTAs of a launch that run at once, `per_sm` to an SM. Clusters of three CTAs and more do not fill the machine (SMs of a GPC stay over).
static long w4_at_once(int per_sm, int cluster, int num_sms) { return (long)per_sm * num_sms * (cluster > 2 ? 7 : 8) / 8; }

// Shares of a row tile's K (logarithms): 2^wk of a CTA's warps, 2^ct CTAs. As many as make the launch 256 CTAs (150 from 17 rows on, where
// a CTA's work per block of K doubles), each share keeping four blocks. Measured (us, asking for 256 / 512 / 1024): 4096 x 4096, 1 row 3.4 /
// 4.3 / 4.3; 6144 x 4096, 1 row 4.4 / 7.2 / 7.2; 28672 x 4096, 1 row 15.3 / 15.2 / 16.5; 14336 x 4096, 8 rows 10.6 / 11.8; 10240 x 5120, 8 rows
// 10.0 / 11.9; 27648 x 5120, 4 rows 16.5 / 18.6 (19.0 asking for 200). 32 rows through 4096 x 4096: 19 with eight warps of a CTA to a tile, 8.7
// with two of each of four.
// Shares go to warps first; to CTAs where a CTA's part of the batch would outweigh its weights (every CTA of a tile reads all of its share
// of the batch) or not fit beside a neighbour's. Joining a cluster costs some 0.7 us, so small batches' short rows stay in a CTA.
// The first: several warps to a tile are fewer tiles to a CTA, and the batch is read that much more often. Measured (us, warps to a tile x CTAs):
// 10240 x 5120 at 4 rows 4 x 1 9.2, 8 x 1 10.3, 1 x 4 8.9, at 8 rows 2 x 2 9.8, 8 x 1 14.2, 1 x 4 9.4, at 16 rows 1 x 4 12.7, 2 x 4 14.7, 8 x 1
// 25.1; 4096 x 4096 at 16 rows 2 x 4 5.2, 1 x 8 6.0, 8 x 1 7.6; below 48 KB 6144 x 4096 at 4 rows 8 x 1 5.0, 2 x 4 5.3. The second, 56 KB (72
// from 17 rows on) of the batch in a CTA: 4096 x 14336 at 16 rows 56 KB 11.5, 112 KB 14.0; 27648 x 5120 at 8 rows 41 KB 17.2, 82 KB 19.5, but
// 28672 x 4096 at 8 33 KB 17.1, 66 KB 15.9; 14336 x 4096 at 32 rows 66 KB 23.0, 132 KB 27.1. Over seven weights at 2 to 32 rows, int4 and e2m1,
// the rule is within a tenth of the best in four cases of five; farthest are 28672 x 4096 at 6 rows of e2m1 (22.7, 1 x 1 17.8), 14336 x 4096 at 4
// of those (12.6, 1 x 2 10.0) and 4096 x 4096 at 32 rows (9.2, 2 x 4 7.5).
static void w4_rows_split(const W4Weight& w, int M, int unit, int num_sms, int& wk, int& ct) {
    const int blocks = w.blocks(), units = blocks / unit, tiles = w.row_tiles(), enough = M > 16 ? 150 : 256;
    int p = 0;                                          // log2 of all shares
    while (p < 6 && ((long)tiles << p) < 8l * enough && (blocks >> (p + 1)) >= 4) ++p;
    const long ctas = ((long)tiles << p) / 8, batch = (long)M * blocks * 128;                // bytes of the batch in a CTA of a whole K
    wk = min(p, 3);
    if (batch >= 48 * 1024 && ctas >= PIE_SMS && M > 2) wk = min(wk, M <= 4 ? 2 : M <= 8 ? 1 : M <= 16 && p >= 3 ? 1 : 0);
    ct = min(p - wk, 3);
    while (ct < 3 && (long)M * w4r_row_bytes(((units - 1 >> ct) + 1) * unit) > (M > 16 ? 72 : 56) * 1024) {
        ++ct;
        if (wk + ct > p && wk > 0) --wk;
    }
    const long all = (long)((tiles + (8 >> wk) - 1) / (8 >> wk)) << ct;
    if (M > 16 && ct > 1 && all > w4_at_once(2, 1 << ct, num_sms) && all <= 2l * num_sms &&                // one round, not two
        (long)M * w4r_row_bytes(((units - 1 >> (ct - 1)) + 1) * unit) <= W4R_BATCH)
        --ct;
    while (wk + ct > 5) --wk;                           // a CTA of the cluster stores four features or more
}

// CTAs per SM of a launch of few rows, of 2 .. most: as few as hold the launch in the least rounds. The scheduler fills an SM before it takes
// the next, so that 256 CTAs of which four fit leave half the SMs idle: 4096 x 14336 at 8 rows 9.0 us with two, 11.6 with three, 13.7 with
// four; 6144 x 4096 (384 CTAs) 8.2 / 5.5 / 6.7; 10240 x 5120 (640) 12.2 / 9.5 / 12.0. Where the rounds are many they even out by themselves, and
// more threads win: 28672 x 4096 (1792) 19.5 / 20.0 / 17.7.
static int w4_rows_resident(long ctas, int cluster, int most, int num_sms) {
    if (ctas >= 8l * num_sms) return most;
    int best = most;
    for (int r = most - 1; r >= 2; --r) {
        const auto work = [&](int n) { return (ctas - 1) / w4_at_once(n, cluster, num_sms) * n + n; };
        if (work(r) < work(best)) best = r;
    }
    return best;
}

template <int KIND, int GROUP, int NT, int RESIDENT>
static cudaError_t launch_w4_rows(const W4Weight& w, const W4Call& c, int wk, int ct, int tiles, int smem) {
    auto kern = w4_rows_kernel<KIND, GROUP, NT, RESIDENT>;
    static std::atomic<unsigned long long> done{0};
    if (smem > 48 * 1024) {
        const cudaError_t e = w4_all_smem(kern, done);
        if (e != cudaSuccess) return e;
    }
    return w4_launch(kern, dim3(tiles << ct), 256, smem, 1 << ct, c.st, w, c.x, c.ldx, c.C, c.ldc, c.R, c.ldr, c.M, c.epi, wk, ct, c.status);
}
template <int KIND, int GROUP>
static cudaError_t launch_w4_rows_nt(const W4Weight& w, const W4Call& c) {
    const int unit = W4R_UNIT<GROUP>, units = w.blocks() / unit, nt = c.M <= 8 ? 1 : c.M <= 16 ? 2 : 4;
    int wk, ct;
    w4_rows_split(w, c.M, unit, c.num_sms, wk, ct);
    const int wr = 8 >> wk, tiles = (w.row_tiles() + wr - 1) / wr;
    int smem = w4r_smem(c.M, ((units - 1 >> ct) + 1) * unit, nt, wr * 16, 1 << ct);
    if (smem > 227 * 1024) return cudaErrorInvalidValue;
    const int resident = w4_rows_resident((long)tiles << ct, 1 << ct, nt == 1 ? 4 : nt == 2 ? 3 : 2, c.num_sms);
    smem = max(smem, 228 * 1024 / (resident + 1) - 1008);                // no more of them fit
    if (nt == 4) return launch_w4_rows<KIND, GROUP, 4, 2>(w, c, wk, ct, tiles, smem);
    if (resident == 2)
        return nt == 1 ? launch_w4_rows<KIND, GROUP, 1, 2>(w, c, wk, ct, tiles, smem) : launch_w4_rows<KIND, GROUP, 2, 2>(w, c, wk, ct, tiles, smem);
    return nt == 1 ? launch_w4_rows<KIND, GROUP, 1, 4>(w, c, wk, ct, tiles, smem) : launch_w4_rows<KIND, GROUP, 2, 3>(w, c, wk, ct, tiles, smem);
}
template <int KIND>
static cudaError_t launch_w4_rows_group(const W4Weight& w, const W4Call& c) {
    return w.group == 32 ? launch_w4_rows_nt<KIND, 32>(w, c) : w.group == 64 ? launch_w4_rows_nt<KIND, 64>(w, c) : launch_w4_rows_nt<KIND, 128>(w, c);
}

// CTAs that share the K of 128 weight rows in the tensor cores' way: the least of the blocks of 64 columns of a CTA and what the join costs in
// blocks, where two CTAs of an SM hold each other up by a third. Measured (us, at 48 rows): 4096 x 14336 45 (1), 28 (2), 21.8 (3), 19.7 (4), 18.4
// (8); 10240 x 5120 19.9 (1), 16.8 (2), 15.1 (3), 22.2 (4: two rounds); 6144 x 4096 12.5 (2), 12.8 (3), 11.4 (4); 5120 x 5120 13.9 (2), 12.5 (3),
// 12.3 (4); 1024 x 8192 12.4 (4), 10.1 (8); 2048 x 8192 12.5 (4), 18.9 (8: two rounds); 14336 x 1024 8.1 (1), 9.1 (2); 4096 x 1024 7.3 (2), 7.2
// (4), of 256 rows 10.9 (2), 12.5 (4). The join of three is set at what leaves them the weights with which four take two rounds.
static int w4_tile_splits(long items, int blocks, int num_sms) {
    int best = 1;
    double least = 0;
    for (const int s : {1, 2, 3, 4, 8}) {
        if (s > 1 && (items * s > w4_at_once(2, s, num_sms) || blocks < 4 * s || (s == 8 && items * 8 > num_sms / 2))) continue;
        const double join = s == 1 ? 0 : s == 3 ? 7.5 : 3 + 0.5 * s, beside = items * s <= w4_at_once(1, s, num_sms) ? 1 : 1.35;
        const double t = ((blocks + s - 1) / s + join) * beside;
        if (s == 1 || t < least) best = s, least = t;
    }
    return best;
}

// Most rows of a batch that runs here. From 9 rows on the expansion's work doubles per eight rows, and from 17 on the MMAs' too, so that a
// product's time grows with its weights, while the tensor cores' way (with the rows' conversion) takes some microseconds and a fifth or a
// quarter of one per block of 64 columns of a CTA's: the smaller of the two lines is taken. Measured, this way against the other (us), at 16
// rows: 4096 x 4096 5.2 / 9.7, 6144 x 4096 7.2 / 10.6, 14336 x 1024 6.0 / 7.2, 10240 x 5120 12.7 / 14.0, 4096 x 14336 11.4 / 17.5, 14336 x 4096
// 14.5 / 14.7, 28672 x 4096 28 / 20.6; at 32: 9.4 / 10.2, 11.6 / 11.2, 7.3 / 7.6, 26 / 14.5, 38 / 18, 23 / 15, 42 / 21. Of e2m1 at 16: 8.0 /
// 9.7, 10.1 / 10.5, 10.5 / 7.2, 15.7 / 14.0, 15.6 / 17.5, 20 / 14.6, 39 / 20. Shared memory of a cluster of eight bounds the batch's share.
PIE_API int pie_gemm_w4_rows(int N, int K, int fp4, int num_sms) {
    const int panels = (N + 127) / 128, blocks = (K + 63) / 64, splits = w4_tile_splits(panels, blocks, num_sms);
    const double weights = 1e-6 * N * K, rounds = splits > 1 ? 1 : (panels + 2 * num_sms - 1) / (2 * num_sms);
    const double block = (long)panels * splits <= w4_at_once(1, splits, num_sms) ? 0.19 : 0.245;
    const double tiles = (splits > 1 ? 7 : 4.5) + block * ((blocks + splits - 1) / splits) * rounds;
    const int most = !fp4 && 3 + 0.37 * weights < tiles ? 32 : (fp4 ? 4 + 0.24 * weights : 3 + 0.19 * weights) < tiles ? 16 : 8;
    return min(most, W4R_BATCH / w4r_row_bytes((K + 1023) / 1024 * 2));
}

// C[M, N] (or [M, N / 2] behind a GLU) = x[M, K] * W^T of up to pie_gemm_w4_rows(N, K) rows.
PIE_API int pie_gemm_w4(const void* weight, const void* x, int ldx, void* C, int ldc, const void* R, int ldr, int M, int epilogue,
                        int* status, int num_sms, cudaStream_t st) {
    const W4Weight& w = *reinterpret_cast<const W4Weight*>(weight);
    const W4Call c{(const bf16*)x, ldx, (bf16*)C, ldc, (const bf16*)R, ldr, M, epilogue, status, num_sms, st};
    if (int e = w4_check(w, c)) return e;
    if (M <= 0) return 0;
    if (M > 32 || w.experts != 1) return (int)cudaErrorInvalidValue;
    const int kind = w4_kind(w);
    const cudaError_t e = kind == W4_FP4 ? launch_w4_rows_group<W4_FP4>(w, c)
                        : kind == W4_ZERO ? launch_w4_rows_group<W4_ZERO>(w, c) : launch_w4_rows_group<W4_INT>(w, c);
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

typedef CUresult (*W4EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// fp16 rows of `blocks` blocks of 64 columns, see W4Maps.
static bool w4_map(CUtensorMap* map, const void* ptr, long rows, int blocks, int box_rows, int box_blocks) {
    static W4EncodeFn enc = nullptr;
    if (!enc) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return false;
        enc = reinterpret_cast<W4EncodeFn>(p);
    }
    if ((uintptr_t)ptr & 15) return false;
    const cuuint64_t dims[3] = {GEMM_BK, (cuuint64_t)rows, (cuuint64_t)blocks}, strides[2] = {(cuuint64_t)blocks * GEMM_BK * 2, GEMM_BK * 2};
    const cuuint32_t box[3] = {GEMM_BK, (cuuint32_t)box_rows, (cuuint32_t)box_blocks}, step[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The rows in fp16 [rows, K padded to 64] and their factors.
struct W4Rows16 {
    void* x;
    float* back;
    long rows;
};

template <int KIND, int GROUP>
static cudaError_t launch_w4_tile(const W4Weight& w, const W4Call& c, const W4Rows16& r, const W4Work& work, int splits, long items) {
    auto kern = w4_tile_kernel<KIND, GROUP>;
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = w4_all_smem(kern, done);
    if (e != cudaSuccess) return e;
    W4Shape shape{work.tile_rows, splits, 0, 0, 0};
    const int budget = 112 * 1024 - 1024 - (int)W4T_BAR_BYTES - 64;          // two CTAs per SM
    // Two blocks per stage of the batch where they are few columns, as each stage costs the MMA issuer a wait and a commit; three stages of
    // codes where that leaves the batch six blocks, which cover a load's way.
    shape.x_blocks = shape.room <= 64 ? 2 : 1;
    const int x_bytes = shape.room * GEMM_BK * 2 * shape.x_blocks, c_bytes = (int)W4T_C_BYTES<KIND, GROUP>;
    auto total = [&](int xs, int cs) { return max(xs * x_bytes, shape.splits > 1 ? (int)w4_join_bytes(shape.room) : 0) + cs * c_bytes; };
    shape.c_stages = total((6 + shape.x_blocks - 1) / shape.x_blocks, 3) <= budget ? 3 : 2;
    shape.x_stages = W4T_X_STAGES;
    while (shape.x_stages > 2 && total(shape.x_stages, shape.c_stages) > budget) --shape.x_stages;
    int smem = total(shape.x_stages, shape.c_stages) + 1024 + (int)W4T_BAR_BYTES + 64;
    W4Maps maps;
    for (int i = 0; i < (work.items ? 4 : 1); ++i)
        if (!w4_map(&maps.x[i], r.x, r.rows, w.blocks(), work.items ? 16 << i : work.tile_rows, shape.x_blocks)) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(splits > 1 ? items * splits : min(items, 2l * c.num_sms)));
    // Where every CTA can have an SM to itself: without room for a second one, which the scheduler would put there (128 rows through 4096
    // x 14336 30.5 -> 24.7 us, 4096 x 4096 15.6 -> 13.3)
    if (grid.x <= w4_at_once(1, splits, c.num_sms)) smem = max(smem, 116 * 1024);
    return w4_launch(kern, grid, W4T_THREADS, smem, splits, c.st, maps, w, r.back, c.C, c.ldc, c.R, c.ldr, work, shape, c.epi, c.status);
}
template <int KIND>
static cudaError_t launch_w4_tile_group(const W4Weight& w, const W4Call& c, const W4Rows16& r, const W4Work& work, int splits, long items) {
    return w.group == 32 ? launch_w4_tile<KIND, 32>(w, c, r, work, splits, items)
         : w.group == 64 ? launch_w4_tile<KIND, 64>(w, c, r, work, splits, items) : launch_w4_tile<KIND, 128>(w, c, r, work, splits, items);
}

// items_at: scratch of int4 [1 + max_mtiles * 8] where there are tiles, else null.
static int w4_tiles(const W4Weight& w, const W4Call& c, const W4Rows16& r, const W4Tiles& tiles, void* items_at) {
    if (int e = w4_check(w, c)) return e;
    const bool sorted = tiles.expert != nullptr;
    if (!r.x || !r.back || (sorted && !items_at)) return (int)cudaErrorInvalidValue;
    W4Work work{(int4*)items_at, c.M, 0};
    int rows_per_tile = 0;                  // blocks of the conversion per 128 rows of a sorted batch
    if (sorted) {
        // About as wide as the experts' rows are on average (the counts are on the device): an expert with more rows takes several items.
        // Measured (us, items of 32 / 64 / 128 rows): 4 of 32 experts of 5760 x 2880, 8 rows each 71 / 71 / 80, 16 82 / 75 / 84, 24 85 / 79 / 86,
        // 32 105 / 87 / 89, 50 130 / 95 / 97; 8 of 128 of 1536 x 2048, 8 rows 58 / 59 / 65, 16 71 / 71 / 75, 25 86 / 75 / 80, 38 104 / 90 / 93.
        const long least = tiles.max_mtiles > w.experts ? (tiles.max_mtiles - w.experts) * (long)GEMM_BM / w.experts : 0;
        work.tile_rows = least <= 8 ? 32 : least <= 24 ? 64 : 128;
        // Some 2500 blocks (us, with 16 / 32 / 64 / 128 per tile: 1500 tokens of 4 of 32 experts 217 / 210 / 209 / 208, 512 of 2 of 8 80 / 69 / 64
        // / 58, 1024 of 8 of 128 122 / 118 / 122 / 127, 128 of those 61 / 62 / 67 / 76)
        rows_per_tile = least <= 8 ? 16 : max(32, min(128, 2560 / (tiles.max_mtiles + 1)));
    } else {
        const int parts = (c.M + 127) / 128;
        work.tile_rows = ((c.M + parts - 1) / parts + 15) / 16 * 16;      // equal shares of the batch
    }
    const int kbs = w.blocks();
    const dim3 grid(sorted ? tiles.max_mtiles + 1 : 1, sorted ? rows_per_tile : min(c.M, 65535));
#define ROWS(VECS) launch_pdl(w4_rows_fp16_kernel<VECS>, grid, dim3(256), 0, c.st, c.x, c.ldx, (__half*)r.x, r.back, w.k, kbs * 64, work, tiles)
    cudaError_t e = w.k <= 2048 ? ROWS(1) : w.k <= 4096 ? ROWS(2) : w.k <= 8192 ? ROWS(4) : ROWS(8);
#undef ROWS
    if (e != cudaSuccess) return (int)e;
    const long items = w.panels() * (sorted ? (long)tiles.max_mtiles * (256 / work.tile_rows) : (c.M + work.tile_rows - 1) / work.tile_rows);
    const int splits = sorted ? 1 : w4_tile_splits(items, kbs, c.num_sms);
    const int kind = w4_kind(w);
    e = kind == W4_FP4 ? launch_w4_tile_group<W4_FP4>(w, c, r, work, splits, items)
      : kind == W4_ZERO ? launch_w4_tile_group<W4_ZERO>(w, c, r, work, splits, items) : launch_w4_tile_group<W4_INT>(w, c, r, work, splits, items);
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

// The same for any number of rows; x16 [M, K padded to 64] fp16 and back [M] are scratch.
PIE_API int pie_gemm_w4_tiles(const void* weight, const void* x, int ldx, void* x16, float* back, void* C, int ldc, const void* R, int ldr,
                              int M, int epilogue, int* status, int num_sms, cudaStream_t st) {
    if (M <= 0) return 0;
    const W4Weight& w = *reinterpret_cast<const W4Weight*>(weight);
    if (w.experts != 1) return (int)cudaErrorInvalidValue;
    const W4Call c{(const bf16*)x, ldx, (bf16*)C, ldc, (const bf16*)R, ldr, M, epilogue, status, num_sms, st};
    return w4_tiles(w, c, W4Rows16{x16, back, M}, W4Tiles{nullptr, nullptr, 0, 1}, nullptr);
}

template <int KIND, int GROUP>
static cudaError_t launch_w4_experts(const W4Weight& w, const W4Call& c, const W4Tiles& tiles) {
    auto kern = w4_experts_kernel<KIND, GROUP>;
    const int smem = w4e_smem(w.blocks());
    if (smem > 227 * 1024) return cudaErrorInvalidValue;
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = w4_all_smem(kern, done);
    if (e != cudaSuccess) return e;
    const int resident = smem <= 113 * 1024 ? 2 : 1;
    return w4_launch(kern, dim3(c.num_sms * resident), 256, smem, 1, c.st, w, c.x, c.ldx, c.C, c.ldc, tiles, c.epi, c.status);
}
template <int KIND>
static cudaError_t launch_w4_experts_group(const W4Weight& w, const W4Call& c, const W4Tiles& tiles) {
    return w.group == 32 ? launch_w4_experts<KIND, 32>(w, c, tiles)
         : w.group == 64 ? launch_w4_experts<KIND, 64>(w, c, tiles) : launch_w4_experts<KIND, 128>(w, c, tiles);
}

// Whether a sorted batch is best taken eight rows at a time (pie_grouped_gemm_w4_few): where experts have up to four on average, as more
// than eight mean a second pass over an expert's weights. Measured against the tensor cores' way (us; tokens of top-k of experts): 1 of 4
// of 32 (e2m1, 5760 x 2880) 15.7 / 21.8, 32 of those 58 / 73, 64 87 / 70; 1 of 2 of 8 (4096 x 4096) 9.1 / 19.8, 16 of those 21 / 23, 32 26 /
// 24; 64 of 8 of 128 (1536 x 2048) 44 / 57, 128 66 / 61.
PIE_API int pie_grouped_gemm_w4_rows(int experts, int K, long rows) {
    return rows <= 4l * experts && w4e_smem((K + 63) / 64) <= 113 * 1024;
}

// Experts, eight rows at a time: arguments as of pie_grouped_gemm_bf16.
PIE_API int pie_grouped_gemm_w4_few(const void* weight, const void* x, int ldx, void* C, int ldc, const int* tile_expert,
                                    const int* tile_list, int max_mtiles, int epilogue, int* status, int num_sms, cudaStream_t st) {
    if (max_mtiles <= 0) return 0;
    const W4Weight& w = *reinterpret_cast<const W4Weight*>(weight);
    if (!tile_expert || w.experts <= 0 || (epilogue != EPI_STORE && epilogue != EPI_SWIGLU)) return (int)cudaErrorInvalidValue;
    const W4Call c{(const bf16*)x, ldx, (bf16*)C, ldc, nullptr, 0, 0, epilogue, status, num_sms, st};
    if (int e = w4_check(w, c)) return e;
    const W4Tiles tiles{tile_expert, tile_list, max_mtiles, w.experts};
    const int kind = w4_kind(w);
    const cudaError_t e = kind == W4_FP4 ? launch_w4_experts_group<W4_FP4>(w, c, tiles)
                        : kind == W4_ZERO ? launch_w4_experts_group<W4_ZERO>(w, c, tiles) : launch_w4_experts_group<W4_INT>(w, c, tiles);
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

// Experts: arguments as of pie_grouped_gemm_bf16; x16 [max_mtiles * 128, K padded to 64], back [max_mtiles * 128] and items
// [1 + max_mtiles * 8][4] are scratch.
PIE_API int pie_grouped_gemm_w4(const void* weight, const void* x, int ldx, void* x16, float* back, int* items, void* C, int ldc,
                                const int* tile_expert, const int* tile_list, int max_mtiles, int epilogue, int* status, int num_sms,
                                cudaStream_t st) {
    if (max_mtiles <= 0) return 0;
    const W4Weight& w = *reinterpret_cast<const W4Weight*>(weight);
    if (!tile_expert || w.experts <= 0 || (epilogue != EPI_STORE && epilogue != EPI_SWIGLU)) return (int)cudaErrorInvalidValue;
    const W4Call c{(const bf16*)x, ldx, (bf16*)C, ldc, nullptr, 0, 0, epilogue, status, num_sms, st};
    return w4_tiles(w, c, W4Rows16{x16, back, (long)max_mtiles * GEMM_BM}, W4Tiles{tile_expert, tile_list, max_mtiles, w.experts}, items);
}
