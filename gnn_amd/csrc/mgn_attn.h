// Shared by the attention kernels (mgn_attn_fwd.hip, mgn_attn_bwd.hip, mgn_attn_few.hip).
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(s_ij) / sum_j exp(s_ij),   s_ij = scale <q_i, k_j> + table[head][lut[place(i, j)]]
//
// over the keys j of query i's own segment that are not masked.  Scores are kept in base 2 (scale and bias times log2 e).
//
// Operand images.  The matrix instruction v_mfma_f32_32x32x16 takes, from lane (i = lane & 31, h = lane >> 5), eight
// consecutive k values of row i.  Keys, values, queries and gradients are laid out once per call as the very 16 bytes each
// lane will feed, in subtiles of 32 tokens of one head, so that the main kernels copy linear memory into LDS and read it
// back linearly (no bank conflicts, no address arithmetic, no padding or masking left to do):
//   image R (contraction over the head's width):  [plane][width / 16][lane][8],  element = x[token i][16 c + 8 h + e]
//   image T (contraction over the 32 tokens):     [plane][2][width / 32][lane][8], element = x[token t(kc, h, e)][32 b + i]
//   (values in the forward pass; the backward pass, which needs most operands both ways, reads image R transposed: tr_read)
// with t = 16 kc + 4 h + e (e < 4), 16 kc + 8 + 4 h + e - 4 (e >= 4): the order in which a lane already holds the scores of
// one column after a product (rows 8 g + 4 h + t), so probabilities go from one product into the next without a shuffle.
// A segment's first subtile in an image is floor(first token / 32) + segment: no two segments share a subtile, and no table
// of tile offsets is needed.  Rows past a segment's end and masked keys are zeros.
//
// Number formats.  bf16: operands as they are.  fp16: one plane, scaled by a power of two as the next.  fp32: two fp16 planes
// x = 2^e (h1 + h2) with the subtile's own e, or the row's where the subtile's rows are far apart in size (residual 2^-22 of the
// value, 2^-25 of the row's largest magnitude), three partial products per product.  The exponents go into constants that each
// product is multiplied with anyway.  Probabilities and dS enter the second products in units that follow their own size: in two
// planes (fp32: what is left is 2^-36 of the largest addend of a sum) or, in the 16-bit types, in one, rounded to half a step of the
// type as the results are (errors of 2.4e-3 where results rounded once have 1.7e-3 in bf16, 2.9e-4 and 2.1e-4 in fp16).  A second plane
// would add half as many products again; it is taken for the probabilities where a bias table is trained (P2, out32), since the
// table's gradient is a sum that cancels.  A weight below 2^-126 of its row's largest is zero.
#pragma once
#include "mgn_device.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum { AT_BF16 = 0, AT_F16 = 1, AT_F32 = 2 };
constexpr float LOG2E = 1.4426950408889634f;
constexpr float F32_MOST = 3.402823466e38f;
constexpr int TOP = 14;                 // operands are scaled to magnitudes below 2^TOP
constexpr int OVER = 4;                  // the running maximum may lag behind by this much (base 2)
constexpr int FAR_EXP = -60;            // a subtile so much smaller than the largest adds nothing in fp16; its shift stops here
constexpr int ATT_TQ = 128;             // queries (or keys, in the key-gradient kernel) of a workgroup: 32 per wave
constexpr int ATT_MAX_SPLITS = 256;
constexpr int ATT_MAX_REACH = 1024;
constexpr int ATT_MAX_BUCKETS = 64;

template <int KIND> constexpr int planes() { return KIND == AT_F32 ? 2 : 1; }

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

template <int KIND>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (KIND == AT_BF16) return mfma32_bf16(a, b, c);
    else return mfma32_f16(a, b, c);
}

template <int KIND>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (KIND == AT_BF16) return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
}

// eight consecutive values as one operand (hi), and for two planes what is left of them (lo)
template <int KIND, bool TWO = KIND == AT_F32>
__device__ __forceinline__ void pack8(const float* v, u32x4& hi, u32x4& lo) {
    float minus;                                              // -1 that is not folded: v - (float)h as one mixed instruction
    asm("v_mov_b32 %0, -1.0" : "=v"(minus));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KIND == AT_F32 || (KIND == AT_F16 && TWO)) {
            const f16x2 a = __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, f16x2);
            const f32x2 b = {__builtin_fmaf((float)a[0], minus, v[2 * i]), __builtin_fmaf((float)a[1], minus, v[2 * i + 1])};
            hi[i] = __builtin_bit_cast(unsigned, a); lo[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(b, f16x2));
        } else if constexpr (TWO) {
            const unsigned a = pack2<KIND>(v[2 * i], v[2 * i + 1]);
            hi[i] = a;
            lo[i] = pack2<KIND>(v[2 * i] - __uint_as_float(a << 16), v[2 * i + 1] - __uint_as_float(a & 0xffff0000u));
        } else {
            hi[i] = pack2<KIND>(v[2 * i], v[2 * i + 1]);
        }
    }
}

// eight consecutive elements of a row as they lie in memory; 16 bytes (32 for fp32), 16-byte aligned
template <int KIND> struct Raw8 {
    u32x4 w[KIND == AT_F32 ? 2 : 1];
    __device__ __forceinline__ void zero() {
        w[0] = u32x4{0, 0, 0, 0};
        if constexpr (KIND == AT_F32) w[1] = w[0];
    }
    __device__ __forceinline__ void load(const void* base, long long off) {
        const u32x4* p = (const u32x4*)((const char*)base + off * (KIND == AT_F32 ? 4 : 2));
        w[0] = p[0];
        if constexpr (KIND == AT_F32) w[1] = p[1];
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned a = w[0][i];                       // a copy: a bit cast of the vector's element takes element 0
            if constexpr (KIND == AT_F32) {
                const unsigned b = w[1][i];
                v[i] = __uint_as_float(a); v[4 + i] = __uint_as_float(b);
            } else if constexpr (KIND == AT_BF16) {
                v[2 * i] = __uint_as_float(a << 16);
                v[2 * i + 1] = __uint_as_float(a & 0xffff0000u);
            } else {
                const f32x2 f = __builtin_convertvector(__builtin_bit_cast(f16x2, a), f32x2);
                v[2 * i] = f[0]; v[2 * i + 1] = f[1];
            }
        }
    }
};

template <int KIND>
__device__ __forceinline__ void load8(const void* base, long long off, float* v) {
    Raw8<KIND> r;
    r.load(base, off);
    r.get(v);
}

template <int KIND>
__device__ __forceinline__ float load1(const void* base, long long off) {
    if constexpr (KIND == AT_F32) return ((const float*)base)[off];
    else if constexpr (KIND == AT_BF16) return __uint_as_float((unsigned)((const unsigned short*)base)[off] << 16);
    else return (float)((const _Float16*)base)[off];
}

template <int KIND>
__device__ __forceinline__ void store4(void* base, long long off, f32x4 v) {
    if constexpr (KIND == AT_F32) *(f32x4*)((float*)base + off) = v;
    else *(u32x2*)((unsigned short*)base + off) = u32x2{pack2<KIND>(v[0], v[1]), pack2<KIND>(v[2], v[3])};
}

// exponent that brings magnitudes up to `top` below 2^TOP (fp16 formats); infinities get the largest
template <int KIND>
__device__ __forceinline__ int scale_exp(float top) {
    if constexpr (KIND == AT_BF16) return 0;
    const int e = (int)((__float_as_uint(top) >> 23) & 0xff) - 127;
    return top == 0.f ? -126 : min(max(e + 1 - TOP, -126), 114);
}

// Exponent of a block of 32 rows as the images' records hold it, and whether some of its rows have one of their own (rows whose
// largest element is less than 2^-APART of the block's): such a row's elements are scaled by it, and what they are multiplied
// into is corrected by the difference, in branches that other blocks do not take.  So an element loses nothing to a large neighbour
// row: its two fp16 terms leave 2^-22 of it, or 2^-25 of its own row's largest element.
constexpr int APART = 14;
__device__ __forceinline__ int block_word(int ex, bool apart) { return (ex & 0xffff) | (apart ? 0x10000 : 0); }
__device__ __forceinline__ int block_exp(int word) { return (int)(short)word; }
__device__ __forceinline__ bool block_apart(int word) { return (word & 0x10000) != 0; }
// differences of the rows 8 q + 4 h .. + 3, q < 4, which a lane's scores belong to
struct RowFix { i32x4 f[4]; };
__device__ __forceinline__ RowFix row_fix(const int* of_block, int h) {
    RowFix r;
#pragma unroll
    for (int q = 0; q < 4; ++q) r.f[q] = *(const i32x4*)(of_block + 8 * q + 4 * h);
    return r;
}
__device__ __forceinline__ void apply_fix(f32x16& s, const RowFix& r) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_ldexpf(s[e], r.f[e >> 2][e & 3]);
}
// 2^e, zero below the smallest number, the largest power of two where it would be infinite
__device__ __forceinline__ float unit_factor(int e) { return __builtin_amdgcn_ldexpf(1.f, min(e, 127)); }

// largest magnitude of N values, infinities left out: they stay what they are under any scaling and set none for their neighbours
template <int N> __device__ __forceinline__ float finite_top(const float (*v)[8]) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, (__float_as_uint(v[c][e]) & 0x7fffffffu) < 0x7f800000u ? fabsf(v[c][e]) : 0.f);
    return top;
}
// The same for a row that lanes l and l + 32 hold half of each; the second pass is taken where there is an infinity.
template <int N> __device__ __forceinline__ float row_top(const float (*v)[8]) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[c][e]));
    if (__any(__float_as_uint(top) >= 0x7f800000u)) top = finite_top<N>(v);
    return fmaxf(top, __shfl_xor(top, 32));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ int attn_dp_device(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// ------------------------------------------------------------------------------------------------ segments
// Offsets are clamped to [0, T] wherever they are read, so wrong ones give wrong results but no access out of bounds.
__device__ __forceinline__ long long seg_at(const int* ptr, int s, int n_seg, long long T) {
    if (!ptr) return s == 0 ? 0 : T;
    const long long v = ptr[s];
    return v < 0 ? 0 : v > T ? T : v;
}

struct Seg { int seg; int local; long long first; int len; };

// segment and tile within it of tile `tile` when every segment s starts at tile floor(first / 2^shift) + s
__device__ __forceinline__ Seg find_tile(const int* ptr, int n_seg, long long T, int shift, int tile) {
    int lo = 0, hi = n_seg;                                   // the last s whose first tile is <= tile
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((seg_at(ptr, mid, n_seg, T) >> shift) + mid <= tile) lo = mid; else hi = mid;
    }
    Seg g;
    g.seg = lo;
    g.first = seg_at(ptr, lo, n_seg, T);
    const long long end = seg_at(ptr, lo + 1, n_seg, T);
    g.len = (int)(end > g.first ? end - g.first : 0);
    g.local = tile - (int)((g.first >> shift) + lo);
    return g;
}

// Rows of a dense or strided output that belong to no segment, set to zero by all workgroups of a launch together.
template <int KIND>
__device__ __forceinline__ void zero_outside(const int* ptr, int n_seg, long long T, void* out, long long st, long long sh, int heads, int dim) {
    const long long lo = seg_at(ptr, 0, n_seg, T), hi = seg_at(ptr, n_seg, n_seg, T), n = lo + (T - hi);
    if (!ptr || n <= 0 || hi < lo) return;
    const int quads = dim / 4;
    for (long long i = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < n * heads * quads;
         i += (long long)gridDim.x * gridDim.y * blockDim.x) {
        const long long r = i / quads / heads, row = r < lo ? r : hi + (r - lo);
        store4<KIND>(out, row * st + i / quads % heads * sh + 4 * (i % quads), f32x4{0.f, 0.f, 0.f, 0.f});
    }
}

// ------------------------------------------------------------------------------------------------ places and buckets
// Index into the bucket table of the key at `k` seen from the query at `q`.
//   line (one axis): k - q held to [-reach, reach], plus reach
//   lattice (two or three axes): the whole part of the Euclidean distance, held to reach.  d2 = dx^2 + dy^2 + dz^2 is exact
//   below 2^24 and only grows beyond, and sqrt(d2 + 1/2) lies at least 1/(4 reach) off every whole number for d2 <= reach^2:
//   with reach <= 1024 that is 4 units in the last place, so the hardware root (1 ulp) gives the exact whole part.
//   Differences saturate, so any places on either side are right: one instruction either way.
template <int AXES>
__device__ __forceinline__ int place(int qx, int qy, int qz, int kx, int ky, int kz, int reach, float most) {
    if constexpr (AXES == 1) {
        return min(max(__builtin_elementwise_sub_sat(kx, qx), -reach), reach) + reach;
    } else {
        const float dx = (float)__builtin_elementwise_sub_sat(kx, qx), dy = (float)__builtin_elementwise_sub_sat(ky, qy);
        float d2 = __builtin_fmaf(dx, dx, 0.5f);
        d2 = __builtin_fmaf(dy, dy, d2);
        if constexpr (AXES == 3) { const float dz = (float)__builtin_elementwise_sub_sat(kz, qz); d2 = __builtin_fmaf(dz, dz, d2); }
        return (int)__builtin_amdgcn_sqrtf(fminf(d2, most));
    }
}

// Places of the four consecutive keys (queries) 8 q + 4 h .. of a subtile laid out [axis][32].
template <int AXES>
__device__ __forceinline__ void places4(const int* p, i32x4& x, i32x4& y, i32x4& z) {
    x = *(const i32x4*)p;
    y = z = x;
    if constexpr (AXES > 1) y = *(const i32x4*)(p + 32);
    if constexpr (AXES > 2) z = *(const i32x4*)(p + 64);
}

// Scores of masked keys to minus infinity.  Called in a branch that is taken where a subtile has masked keys; the opaque copy of
// the bits keeps it one (the compiler would otherwise test all 16 bits in every step: a third of its vector instructions).
__device__ __forceinline__ void mask_scores(f32x16& s, int valid, int h) {
    unsigned bits = (unsigned)valid >> (4 * h);
    asm volatile("" : "+v"(bits));
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (!(bits >> (8 * (e >> 2) + (e & 3)) & 1)) s[e] = -__builtin_inff();
}

// Where a NaN decides something it is looked for in its bits, which the compiler must not take for a float's: some of these files
// are compiled without regard for NaN in maxima and comparisons (see build.py), and it turns tests of bits into such comparisons.
__device__ __forceinline__ unsigned magnitude_bits(float x) {
    unsigned b = __float_as_uint(x) & 0x7fffffffu;
    asm("" : "+v"(b));
    return b;
}
__device__ __forceinline__ bool finite_bits(float x) { return magnitude_bits(x) < 0x7f800000u; }
__device__ __forceinline__ bool zero_bits(float x) { return magnitude_bits(x) == 0; }
// 1 / l of a softmax's sum; 0 for a row without keys; NaN where a score was NaN or overflowed
__device__ __forceinline__ float inverse_sum(float l) { return zero_bits(l) ? 0.f : 1.0f / l; }

// Sums of probabilities times values in fp16 formats: kept in units of 2^unit (relative to 2^m, m the running maximum), where unit
// follows the largest (probability x size of its values) so far, as m follows the scores.  (One large value that weighs nothing
// must not push all other probabilities into the smallest numbers of fp16.)  A block's probabilities enter times 2^(ev - unit), ev its
// values' exponent.  `unit` is any real number: what rounds in it is made up for in the factor that the sums so far are scaled with.
constexpr float SUM_UNIT_LEAST = -200.f;
// Raises the maximum to the scores' `top` and scales *l, the sum of exponentials; returns how far the old maximum lies below (<= 0).
__device__ __forceinline__ float raise_max(float& m, float& l, float top) {
    const float mn = fmaxf(m, top), lowered = m - (mn == -__builtin_inff() ? 0.f : mn);
    l *= __builtin_amdgcn_exp2f(lowered);
    if (mn > 0.f && !finite_bits(mn)) asm("v_mov_b32 %0, 0x7fc00000" : "=v"(l));      // a score overflowed: no softmax
    m = mn;
    return lowered;
}
// Raises the unit to `need`, the largest (probability x size of its values) of a block, log 2 and relative to 2^m; returns the factor
// for the sums so far.
__device__ __forceinline__ float raise_unit(float& unit, float lowered, float need) {
    const float to = fmaxf(fmaxf(unit + lowered, need), SUM_UNIT_LEAST), by = __builtin_amdgcn_exp2f(lowered + (unit - to));
    unit = to;
    return by;
}
// ACC: the sums stay in accumulation registers, where the products keep them.  (The compiler gives plain multiplications in this
// rare branch a second copy of all of them and then spills: dK and dV of 8192 x 4096, 8 heads of 128, fp32, whole backward pass
// 1683 instead of 1452 us.)  What a product wrote may be read 19 cycles after it was issued, and read by a product 2 after it was
// written: the waits are in the statement.
template <bool ACC> __device__ __forceinline__ void scale16(f32x16& s, float by) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        if constexpr (ACC) {
            float x = s[e], t;
            if (e == 0) asm volatile("s_nop 15\n\ts_nop 7\n\tv_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %2, %1\n\tv_accvgpr_write_b32 %0, %1\n\ts_nop 3" : "+a"(x), "=&v"(t) : "v"(by));
            else asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %2, %1\n\tv_accvgpr_write_b32 %0, %1\n\ts_nop 3" : "+a"(x), "=&v"(t) : "v"(by));
            s[e] = x;
        } else {
            s[e] *= by;
        }
    }
}
// x 2^e for a real e
__device__ __forceinline__ float scale_real(float x, float e) {
    const float whole = rintf(e);
    return ldexpf(x * __builtin_amdgcn_exp2f(e - whole), (int)whole);
}

// What the products of two scaled operands are multiplied with.  Held to normal numbers: with two blocks of zeros it would be zero,
// and minus infinity, the score of a masked key, times zero is no number.
__device__ __forceinline__ float score_factor(float c) { return fminf(fmaxf(c, 0x1p-126f), F32_MOST); }

__device__ __forceinline__ float bias_log2(float b) {          // finite biases stay finite in base 2
    const float v = b * LOG2E;
    return finite_bits(b) ? fminf(fmaxf(v, -F32_MOST), F32_MOST) : v;
}

// ------------------------------------------------------------------------------------------------ copies into LDS
// A zero the compiler knows nothing of: an address plus this is one per lane, so what is loaded from it stays in vector
// registers until it is asked for.  (A load from a uniform address is moved into a scalar register where it is issued -- with a
// wait for the whole memory latency.)
__device__ __forceinline__ int lane_zero() {
    int z;
    asm("v_mov_b32 %0, 0" : "=v"(z));
    return z;
}

// Image R in LDS, read both ways.  Operand T (contraction over the tokens): lane (i, h) gets x[token t(kc, h, e)][32 b + i], see
// above, by two transposing reads, each of four tokens' 16-element chunks.  Four of the chunks that 32 lanes read lie whole multiples
// of 512 bytes apart, in the same banks; so token groups of four are stored rotated, group n of (chunk c, half h) at n ^ (h + 2 (c & 1)),
// which spreads them over all 64 banks and costs no instruction in a step (both offsets below are a lane's own).
// Byte offset of lane (i, h)'s 16 bytes within a chunk of 1 KB:
__device__ __forceinline__ int rot_lane(int lane, int odd) {
    const int h = lane >> 5;
    return h * 512 + (((lane & 31) * 16) ^ (64 * (h + 2 * odd)));
}
template <int NC>
__device__ __forceinline__ u32x4 rot_read(const unsigned short* image, int even, int odd, int plane, int c) {
    return *(const u32x4*)((const char*)image + ((c & 1 ? odd : even) + (plane * NC + c) * 1024));
}
__device__ __forceinline__ int tr_lane(int lane) {             // bytes, tokens 0 .. 3 (+ 8 at this ^ 128)
    const int r = lane >> 2 & 3, s = lane & 3, g = lane >> 4 & 1;
    return g * 1024 + (s >> 1) * 512 + ((64 * (lane >> 5) + 16 * r) ^ (64 * ((s >> 1) + 2 * g))) + (s & 1) * 8;
}
template <int DP>
__device__ __forceinline__ u32x4 tr_read(const unsigned short* image, int at, int plane, int kc, int b) {
    const char* p = (const char*)image + (plane * 64 * DP + b * 2048 + kc * 256);
    const u32x2 lo = lds_tr4((const unsigned short*)(p + at)), hi = lds_tr4((const unsigned short*)(p + (at ^ 128)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Exponents and valid bits of a step (key exponent, value exponent, mask), requested a step ahead and then made uniform.  Only
// what is used is loaded: the unused part of a wider load would be overwritten early, behind a wait for the load.
template <int KIND, int N = 3> struct Record {
    int v[N];
    __device__ __forceinline__ void request(const i32x4* at) {
        const int* p = (const int*)at;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = KIND != AT_BF16 || e == 2 ? p[e] : 0;
    }
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = __builtin_amdgcn_readfirstlane(v[e]);
    }
};

// Linear 1 KB pieces of images on their way into LDS, by way of registers: requested at the top of a step, written at its end.
// (Copies that go straight into LDS would save the registers, but the compiler waits for all of them before the next read
// of ANY shared memory, which put the whole memory latency into every step: 8192 x 8192 at width 128, bf16, 301 us.)
template <int PIECES, int NW = 4> struct Staged {
    static constexpr int N = (PIECES + NW - 1) / NW;          // of each wave
    u32x4 v[N];
    template <typename F> __device__ __forceinline__ void request(int w, int lane, F source) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (PIECES % NW == 0 || NW * n + w < PIECES) v[n] = *(const u32x4*)(source(NW * n + w) + lane * 16);
    }
    __device__ __forceinline__ void write(void* dst, int w, int lane) const { write_at(dst, w, lane * 16); }
    __device__ __forceinline__ void write_rotated(void* dst, int w, int lane) const {
        static_assert(NW % 2 == 0, "a wave's pieces are all even or all odd chunks");
        write_at(dst, w, rot_lane(lane, w & 1));
    }
    __device__ __forceinline__ void write_at(void* dst, int w, int off) const {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (PIECES % NW == 0 || NW * n + w < PIECES) *(u32x4*)((char*)dst + (NW * n + w) * 1024 + off) = v[n];
    }
};

// ------------------------------------------------------------------------------------------------ operand images
struct ImageJob {
    const void* x; long long st, sh;             // rows: element strides of tokens and heads
    const int* ptr; const uint8_t* mask;
    long long T; int heads, n_sub, first_unit;   // n_sub: subtiles of a head; units of this job start at first_unit
    unsigned short* R; unsigned short* Tt;       // images (either may be null; Tt only where ImageArgs::transposed)
    int* ex; int* valid;                         // block word of (head, subtile), 4 ints apart; valid bits of the tokens
    int* fix;                                    // [head][subtile][32]: a row's exponent less the block's (fp16 formats)
    const int* pos; int* pos_out; int axes;      // places [T][axes] -> [subtile][axes][32]
    const void* o; long long o_st, o_sh;         // gradient job: the outputs (fp32 or the type of the rows), ...
    int o_f32;
    int alternate;                               // negate odd subtiles (see mgn_attn_bwd.hip)
    const float* stats; float* rows;             // rows: [head][subtile][3][32] = maximum, 1/sum (fp32: 1), <do, o> (fp32: / sum)
};
struct ImageArgs { ImageJob job[4]; int n_job, units, n_seg, dim, transposed; };

}  // namespace

int mgn_attn_launch_images(int kind, int dp, const void* args, void* stream);     // mgn_attn_fwd.hip
