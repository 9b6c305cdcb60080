// Attention of one set of states over another, backwards.  With P the probabilities and dO the output's gradient:
//   dV = P^T dO,  dP = dO V^T,  dS = P o (dP - <dO_i, o_i>),  dQ = scale dS K,  dK = scale dS^T Q,
//   dtable[head][b] = sum of dS over the pairs in bucket b.
// P is recomputed from the scores and the row statistics of the forward pass.  Two kernels, one that owns queries (dQ and the
// table) and one that owns keys (dK, dV): seven products instead of the five that are needed, but no atomics, so every sum has
// a fixed order and two runs agree bit for bit.
//
// The table's gradient sums dS over very many pairs, and every row of dS sums to zero: an error that all entries share grows
// with their number where the sum itself cancels.  Two such errors are kept out.  The fp16 matrix instruction rounds its sums
// downwards, so dP comes out low everywhere (a 1e-5 error of the table at 20 000 queries): the values' images of odd subtiles
// are negated, dP of those comes out high, and what is left has either sign (6e-7).  And <dO_i, o_i> has to be made of outputs
// that were not rounded to 16 bits: the forward pass keeps them in fp32 where a table is trained (out32).
#include "mgn_attn_host.h"

#include <atomic>

namespace {

struct AttnBwd {
    const int *q_ptr, *k_ptr; long long n_q, n_k; int n_seg, heads, kv_heads, dim; float c0, scale;
    const unsigned short *q_r, *g_r;                   // images R of queries and output gradients, [heads][ns_q]
    const unsigned short *k_r, *v_r;                   // of keys and values, [kv_heads][ns_k]
    const i32x4 *rec_q, *rec_k;                        // exponents {q, g} and {k, v, valid keys}
    const int *fix_q, *fix_g, *fix_k, *fix_v;          // rows' own exponents, [heads][subtile][32]
    const float* rows;                                 // [heads][ns_q][3][32]
    int ns_q, ns_k;
    const int *qpos, *kpos;                            // places [subtile][axes][32]
    const float* table; const int* lut; int n_bucket, reach, axes;
    void *dq, *dk, *dv;                                // dense [tokens][heads][dim]
    double* tpart; float* dtable; int q_tiles;         // [q_tiles][splits][heads][n_bucket]
    int splits; float* part;                           // key side: [split][2][kv_heads][ns_k][32][DP]
    int q_splits; float* q_part;                       // query side: [split][heads][ns_q][32][DP]
    int zero;                                          // rows outside all segments become zeros
    u32x4 *by_query, *by_key;                          // buckets of the pairs, a byte each: [ns_q][ns_k] and [ns_k][ns_q] x [64 lanes][16]
};
constexpr int LISTED = 4;                              // a bias whose buckets are read from there; 1 .. 3: places of so many axes

// Sums in units of 2^unit that follow what is added to them (fp16 formats).  An addend x of a block with exponent ex enters as
// x 2^(ex - unit); one that would pass UNIT_OVER raises the unit to where the largest lies below 2^UNIT_TOP, so that a few that
// grow slowly do not raise it every time and the smallest numbers of fp16 stay 2^-36 of it away.  The factor is one power of two, so
// a block of large exponent raises the unit as well; the first one does.
constexpr int UNIT_LEAST = -1000, UNIT_TOP = 12, FACTOR_MOST = 126;
constexpr float UNIT_OVER = 0x1p15f;
__device__ __forceinline__ int raised_unit(int unit, float most, int ex) {
    return max(max(unit, ex - FACTOR_MOST), (int)((__float_as_uint(most) >> 23) & 0xff) - 126 + ex - UNIT_TOP);
}
__device__ __forceinline__ float largest16(const f32x16& s) {
    float m = fmaxf(fabsf(s[0]), fabsf(s[1]));
#pragma unroll
    for (int e = 2; e < 16; e += 2) m = fmaxf(m, fmaxf(fabsf(s[e]), fabsf(s[e + 1])));
    return m;
}

// A place's bias, base 2, and the byte offset of its bucket's sums.
struct Entry { float bias; int offset; };
// Entries by bucket reach over all values a list can hold.
template <int BIAS> __host__ __device__ constexpr int entries(int reach) { return BIAS == LISTED ? ATT_MAX_BUCKETS : BIAS == 1 ? 2 * reach + 1 : reach + 1; }
template <int BIAS> constexpr int LUTS = entries<BIAS>(ATT_MAX_REACH);
template <int BIAS>
__device__ __forceinline__ int bucket_at(const AttnBwd& a, int r) { return min(max(BIAS == LISTED ? r : a.lut[r], 0), a.n_bucket - 1); }
template <int BIAS>
__device__ __forceinline__ void fill_entries(Entry* entry, const AttnBwd& a, int head, int stride, int t) {
    for (int r = t; r < entries<BIAS>(a.reach); r += 256) {
        const int b = bucket_at<BIAS>(a, r);
        entry[r] = {bias_log2(a.table[head * a.n_bucket + b]), b * stride};
    }
}
template <int BIAS>
__device__ __forceinline__ void fill_biases(float* lutb, const AttnBwd& a, int head, int t) {
    for (int r = t; r < entries<BIAS>(a.reach); r += 256)
        lutb[r] = bias_log2(a.table[head * a.n_bucket + bucket_at<BIAS>(a, r)]);
}
// Buckets of all pairs of a segment, once for all heads and both kernels, as lists of 16 bytes per lane in the order in which each
// kernel's lanes hold a subtile's scores: a lane of the query side 16 keys of its query, of the key side 16 queries of its key.  A
// wave takes one subtile of queries and every gridDim.y-th subtile of keys.  Bound by the vector unit and the two writes: 20 000 x
// 2501, 23 us, 102 MB, 4.4 TB/s; it spares dQ and the table 75 us and dK, dV 25 us of 300 and 285 with four heads.
template <int BIAS>
__global__ __launch_bounds__(256) void attn_buckets_kernel(AttnBwd a) {
    __shared__ unsigned char lutb[LUTS<BIAS>];
    __shared__ __attribute__((aligned(16))) unsigned cross[4][32 * 9];
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    for (int r = t; r < entries<BIAS>(a.reach); r += 256) lutb[r] = (unsigned char)bucket_at<BIAS>(a, r);
    __syncthreads();
    const int qsub = blockIdx.x * 4 + w;
    if (qsub >= a.ns_q) return;
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, 5, qsub);
    if (g.local < 0 || 32 * g.local >= g.len) return;
    const long long k0 = seg_at(a.k_ptr, g.seg, a.n_seg, a.n_k), k1 = seg_at(a.k_ptr, g.seg + 1, a.n_seg, a.n_k);
    const int n_sub = k1 > k0 ? (int)((k1 - k0 + 31) >> 5) : 0;
    const long long kplace = (k0 >> 5) + g.seg;
    const int* qp = a.qpos + (long long)qsub * (BIAS * 32) + j;
    const int qx = qp[0], qy = BIAS > 1 ? qp[32] : 0, qz = BIAS > 2 ? qp[64] : 0;
    const float most = (float)(a.reach * a.reach) + 0.5f;
    unsigned* row = cross[w] + j * 9;
    for (int s = blockIdx.y; s < n_sub; s += gridDim.y) {
        u32x4 list;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            i32x4 x, y, z;
            places4<BIAS>(a.kpos + (kplace + s) * (BIAS * 32) + 8 * q + 4 * h, x, y, z);
            unsigned v = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) v |= (unsigned)lutb[place<BIAS>(qx, qy, qz, x[e], y[e], z[e], a.reach, most)] << (8 * e);
            list[q] = v;
            row[2 * q + h] = v;
        }
        a.by_query[((long long)qsub * a.ns_k + kplace + s) * 64 + lane] = list;
        __builtin_amdgcn_wave_barrier();                       // the wave's own LDS: in order
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned v = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) v |= (unsigned)((const unsigned char*)(cross[w] + (8 * q + 4 * h + e) * 9))[j] << (8 * e);
            list[q] = v;
        }
        a.by_key[((kplace + s) * a.ns_q + qsub) * 64 + lane] = list;
        __builtin_amdgcn_wave_barrier();
    }
}
constexpr int GROUP = 2;                               // sums by bucket that are read, added to and written together

// ------------------------------------------------------------------------------------------------ query side
// A workgroup: 128 queries of one head, 32 per wave, against the key subtiles of its split; two images a step, requested a step ahead
// into registers and read both as they are and transposed.  A lane owns a query: its statistics are registers, and its sums of dS by bucket a column of LDS that no
// other lane touches, two entries read, added to and written at a time (adding the second to the first where both are one bucket;
// readout of 20 000 x 2501 in us for 1 / 2 / 4 / 8 at a time: 753 / 741 / 744 / 771, without the sums 684, before buckets were listed).
//
// Bound by the vector unit with a bias (18 products a step beside about 260 vector instructions with listed buckets, 390
// without): 20 000 x 2501, 4 heads of 32, fp32, plane, table trained, 179 us and 7 for the sum of its two pieces.  Without one by
// the latency of a step's chain: 17 973 x 12 870 in 16 segments, 8 heads of 64, bf16, 75 us = 0.63 PFLOP/s.
template <int KIND, int DP, int BIAS>
__global__ __launch_bounds__(256, DP == 128 && (KIND == AT_F32 || BIAS > 0) ? 1 : KIND == AT_F32 && DP == 32 && BIAS > 0 ? 3 : 2) void attn_dq_kernel(AttnBwd a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, NB = DP / 32, SUB = PL * 32 * DP;
    // fp32 with a bias: one buffer and a second barrier, since two would leave the sums by bucket no room (8192 x 4096, 8 heads of
    // 64: 1095 -> 1028 us for the whole backward pass).  16-bit types: two (8 heads of 32, bf16: 476 us with one, 436 with two).
    constexpr int AXES = BIAS == LISTED ? 0 : BIAS;
    constexpr int BUFS = KIND == AT_F32 && BIAS > 0 ? 1 : 2;
    __shared__ __attribute__((aligned(1024))) unsigned short buf[BUFS][2 * SUB];  // K, V
    __shared__ __attribute__((aligned(16))) int pbuf[AXES ? BUFS : 1][AXES ? 128 : 1];
    extern __shared__ Entry entry[];                                                   // by place, ...
    float* hist = (float*)(entry + entries<BIAS>(a.reach));                            // ... and [4 waves][n_bucket][64], with a table gradient

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.heads, kvh = head / (a.heads / a.kv_heads), tile = blockIdx.x / a.heads, split = blockIdx.y;
    if (a.zero) zero_outside<KIND>(a.q_ptr, a.n_seg, a.n_q, a.dq, (long long)a.heads * a.dim, a.dim, a.heads, a.dim);
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, 7, tile);
    const bool live = g.local >= 0 && g.local * ATT_TQ < g.len;
    if (!live) {
        if (BIAS > 0 && a.tpart && t < a.n_bucket) a.tpart[(((long long)tile * a.q_splits + split) * a.heads + head) * a.n_bucket + t] = 0.0;
        return;
    }
    const long long k0 = seg_at(a.k_ptr, g.seg, a.n_seg, a.n_k), k1 = seg_at(a.k_ptr, g.seg + 1, a.n_seg, a.n_k);
    const int all_sub = k1 > k0 ? (int)((k1 - k0 + 31) >> 5) : 0, per = (all_sub + a.q_splits - 1) / a.q_splits;
    const int s0 = min(split * per, all_sub), n_sub = min(s0 + per, all_sub) - s0;   // this workgroup's share of the key subtiles
    const long long kplace = (k0 >> 5) + g.seg + s0, ksub = (long long)kvh * a.ns_k + kplace;
    const i32x4* rec = a.rec_k + ksub;
    const int qi = g.local * ATT_TQ + 32 * w + j, nsq = (g.len + 31) >> 5;
    const bool mine = qi < g.len;
    const long long row = g.first + min(qi, g.len - 1);
    const long long qsub = (long long)head * a.ns_q + (g.first >> 5) + g.seg + min(g.local * 4 + w, nsq - 1);

    constexpr int PIECES = SUB * 2 / 1024;
    const int last = n_sub - 1, lz = lane_zero(), tl = tr_lane(lane), even = rot_lane(lane, 0), odd = rot_lane(lane, 1);
    Staged<2 * PIECES> st;
    int sp = 0;
    u32x4 listed{}, listed_next{};
    const long long qplace = (g.first >> 5) + g.seg + min(g.local * 4 + w, nsq - 1);
    const u32x4* lists = BIAS == LISTED ? a.by_query + (qplace * a.ns_k + kplace) * 64 + lane : nullptr;
    auto request = [&](int s) {
        st.request(w, lane, [&](int c) {
            const int image = c / PIECES;
            return (const char*)(image == 0 ? a.k_r : a.v_r) + (ksub + s) * (SUB * 2) + (c % PIECES) * 1024;
        });
        if (AXES > 0 && t < AXES * 32) sp = a.kpos[(kplace + s) * (AXES * 32) + t];
        if constexpr (BIAS == LISTED) listed_next = lists[(long long)s * 64];
    };
    auto arrive = [&](int b) {
        st.write_rotated(buf[b], w, lane);
        if (AXES > 0 && t < AXES * 32) pbuf[b][t] = sp;
        listed = listed_next;
    };
    if (n_sub > 0) request(0);

    u32x4 qf[PL][NC], gf[PL][NC];
    {
        const u32x4 *qp = (const u32x4*)(a.q_r + qsub * SUB) + lane, *gp = (const u32x4*)(a.g_r + qsub * SUB) + lane;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int c = 0; c < NC; ++c) { qf[p][c] = qp[(p * NC + c) * 64]; gf[p][c] = gp[(p * NC + c) * 64]; }
    }
    const i32x4 rq = a.rec_q[qsub];
    int eq = 0, eg = 0;                                       // exponents of this query and its gradient
    if constexpr (KIND != AT_BF16) { eq = block_exp(rq[0]) + a.fix_q[qsub * 32 + j]; eg = block_exp(rq[1]) + a.fix_g[qsub * 32 + j]; }
    const float* rp = a.rows + qsub * 96;
    const float m = mine ? rp[j] : __builtin_inff(), norm = KIND == AT_F32 ? 1.f : rp[32 + j], delta = mine ? rp[64 + j] : 0.f;
    int qx = 0, qy = 0, qz = 0;
    float most = 0.f;
    if constexpr (BIAS > 0) {
        if constexpr (AXES > 0) {
            const int* p = a.qpos + qplace * (AXES * 32) + j;
            qx = p[0];
            if (AXES > 1) qy = p[32];
            if (AXES > 2) qz = p[64];
        }
        most = (float)(a.reach * a.reach) + 0.5f;
        fill_entries<BIAS>(entry, a, head, 256, t);
        if (a.tpart)
            for (int r = t; r < a.n_bucket * 256; r += 256) hist[r] = 0.f;
    }
    // Exponent of this query's sums in the second product: dS enters scaled by it and is held below UNIT_OVER.  It follows the dS
    // that actually come (their sizes differ by many orders between queries, and with the keys' weights), as the maximum of a
    // softmax does: when one does not fit, it rises and the sums so far are scaled down.
    int unit = UNIT_LEAST;
    char* sums = (char*)(hist + w * a.n_bucket * 64 + lane);   // this lane's sums of dS by bucket
    Record<KIND> r, rn;
    if (n_sub > 0) { r.request(rec + lz); r.settle(); arrive(0); }

    f32x16 dq[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) dq[b] = zero16();
    __syncthreads();
    for (int sub = 0; sub < n_sub; ++sub) {
        const int b = BUFS == 2 ? sub & 1 : 0;
        request(min(sub + 1, last));
        rn.request(rec + min(sub + 1, last) + lz);
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const u32x4 k1 = rot_read<NC>(buf[b], even, odd, 0, c), v1 = rot_read<NC>(buf[b] + SUB, even, odd, 0, c);
            if constexpr (PL == 2) {
                s = mma<KIND>(rot_read<NC>(buf[b], even, odd, 1, c), qf[0][c], s);
                dp = mma<KIND>(rot_read<NC>(buf[b] + SUB, even, odd, 1, c), gf[0][c], dp);
                s = mma<KIND>(k1, qf[PL - 1][c], s);
                dp = mma<KIND>(v1, gf[PL - 1][c], dp);
            }
            s = mma<KIND>(k1, qf[0][c], s);
            dp = mma<KIND>(v1, gf[0][c], dp);
        }
        int off[BIAS ? 16 : 1];                                // of the buckets' sums
        float add[BIAS ? 16 : 1];
        if constexpr (BIAS > 0)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                i32x4 x, y, z;
                if constexpr (AXES > 0) places4<AXES>(pbuf[b] + 8 * q + 4 * h, x, y, z);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int at;
                    if constexpr (AXES > 0) at = place<AXES>(qx, qy, qz, x[e], y[e], z[e], a.reach, most);
                    else at = listed[q] >> (8 * e) & (ATT_MAX_BUCKETS - 1);
                    const Entry en = entry[at];
                    add[4 * q + e] = en.bias; off[4 * q + e] = en.offset;
                }
            }
        const float c = KIND == AT_BF16 ? a.c0 : score_factor(ldexpf(a.c0, block_exp(r.v[0]) + eq));
        const float up = KIND == AT_BF16 ? 1.f : (s0 + sub) & 1 ? -unit_factor(block_exp(r.v[1]) + eg) : unit_factor(block_exp(r.v[1]) + eg);
        const bool apart = KIND != AT_BF16 && block_apart(r.v[0] | r.v[1]);
        if (r.v[2] != -1 || apart) {
            if (apart) {                                       // rows with exponents of their own
                apply_fix(s, row_fix(a.fix_k + (ksub + sub) * 32, h));
                apply_fix(dp, row_fix(a.fix_v + (ksub + sub) * 32, h));
            }
            mask_scores(s, r.v[2], h);
        }
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            const float x = BIAS > 0 ? __builtin_fmaf(s[n], c, add[BIAS ? n : 0]) - m : __builtin_fmaf(s[n], c, -m);
            const float d = KIND == AT_BF16 ? dp[n] - delta : __builtin_fmaf(dp[n], up, -delta);
            s[n] = __builtin_amdgcn_exp2f(x) * d;                  // dS times this query's sum of exponentials
        }
        if constexpr (BIAS > 0)
            if (a.tpart)
#pragma unroll
                for (int n = 0; n < 16; n += GROUP) {
                    float v[GROUP];
#pragma unroll
                    for (int e = 0; e < GROUP; ++e) v[e] = *(const float*)(sums + off[n + e]);
#pragma unroll
                    for (int e = 0; e < GROUP; ++e) {
#pragma unroll
                        for (int p = 0; p < e; ++p) v[e] = off[n + e] == off[n + p] ? v[p] : v[e];
                        v[e] = __builtin_fmaf(s[n + e], norm, v[e]);
                    }
#pragma unroll
                    for (int e = 0; e < GROUP; ++e) *(float*)(sums + off[n + e]) = v[e];
                }
        if constexpr (KIND != AT_BF16) {
            if (block_apart(r.v[0])) apply_fix(s, row_fix(a.fix_k + (ksub + sub) * 32, h));
            const float most = largest16(s);
            const int ek = block_exp(r.v[0]);
            float f = ldexpf(1.f, ek - unit);
            if (__any(ek - unit > FACTOR_MOST || most * f > UNIT_OVER)) {                     // the two halves of a query's keys only meet here
                const int to = raised_unit(unit, fmaxf(most, __shfl_xor(most, 32)), ek);
                const float by = unit_factor(unit - to);
#pragma unroll
                for (int n = 0; n < NB; ++n) scale16<DP == 128>(dq[n], by);
                unit = to;
                f = ldexpf(1.f, ek - unit);
            }
#pragma unroll
            for (int n = 0; n < 16; ++n) s[n] *= f;
        }
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = s[8 * kc + e];
            u32x4 hi, lo;
            pack8<KIND>(v, hi, lo);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const u32x4 k1 = tr_read<DP>(buf[b], tl, 0, kc, n);
                if constexpr (PL == 2) {
                    dq[n] = mma<KIND>(tr_read<DP>(buf[b], tl, 1, kc, n), hi, dq[n]);
                    dq[n] = mma<KIND>(k1, lo, dq[n]);
                }
                dq[n] = mma<KIND>(k1, hi, dq[n]);
            }
        }
        if (BUFS == 1) __syncthreads();
        arrive(BUFS == 2 ? b ^ 1 : 0);
        r = rn;
        r.settle();
        __syncthreads();
    }
    if (mine) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * n + 8 * q + 4 * h;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = dq[n][4 * q + e] * (a.scale * norm);
                    v[e] = KIND == AT_BF16 ? x : ldexpf(x, unit);
                }
                if (d >= a.dim) continue;
                if (a.q_splits > 1) *(f32x4*)(a.q_part + (((long long)split * a.heads * a.ns_q + qsub) * 32 + j) * DP + d) = v;
                else store4<KIND>(a.dq, (row * a.heads + head) * a.dim + d, v);
            }
    }
    if constexpr (BIAS > 0) {
        if (a.tpart) {
            __syncthreads();
            for (int b = w; b < a.n_bucket; b += 4) {          // one wave sums a bucket's 256 columns, in a fixed order
                double v = 0.0;
#pragma unroll
                for (int x = 0; x < 4; ++x) v += (double)hist[(x * a.n_bucket + b) * 64 + lane];
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
                if (lane == 0) a.tpart[(((long long)tile * a.q_splits + split) * a.heads + head) * a.n_bucket + b] = v;
            }
        }
    }
}

// dtable[head][b] = sum over the query tiles, one wave per entry, fixed order
__global__ __launch_bounds__(64) void attn_table_kernel(const double* __restrict__ part, float* __restrict__ out, int tiles, int entries) {
    const int e = blockIdx.x, lane = threadIdx.x;
    double v = 0.0;
    for (int i = lane; i < tiles; i += 64) v += part[(long long)i * entries + e];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_down(v, o);
    if (lane == 0) out[e] = (float)v;
}

// ------------------------------------------------------------------------------------------------ key side
// A workgroup: 128 keys of one key head, 32 per wave, against its share of the (query head, query subtile) pairs that read
// them.  Here the lane owns a key: rows of the products are queries, whose statistics come through LDS.
// Bound like the query side.  Measured at its two problems: 204 us (fp32, plane, listed buckets, 24 products a step)
// and 100 us = 0.63 PFLOP/s (bf16, four query heads to a key head).
template <int KIND, int DP, int BIAS>
__global__ __launch_bounds__(256, DP == 128 ? 1 : 2) void attn_dkv_kernel(AttnBwd a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, NB = DP / 32, SUB = PL * 32 * DP;
    __shared__ __attribute__((aligned(1024))) unsigned short buf[2][2 * SUB];          // Q, dO
    __shared__ __attribute__((aligned(16))) float rbuf[2][128];
    constexpr int AXES = BIAS == LISTED ? 0 : BIAS;
    __shared__ __attribute__((aligned(16))) int pbuf[AXES ? 2 : 1][AXES ? 128 : 1];
    __shared__ float lutb[BIAS ? LUTS<BIAS> : 1];                                      // the bias by place, of the current head

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x % a.kv_heads, rep = a.heads / a.kv_heads, split = blockIdx.y;
    if (a.zero) {
        zero_outside<KIND>(a.k_ptr, a.n_seg, a.n_k, a.dk, (long long)a.kv_heads * a.dim, a.dim, a.kv_heads, a.dim);
        zero_outside<KIND>(a.k_ptr, a.n_seg, a.n_k, a.dv, (long long)a.kv_heads * a.dim, a.dim, a.kv_heads, a.dim);
    }
    const Seg g = find_tile(a.k_ptr, a.n_seg, a.n_k, 7, blockIdx.x / a.kv_heads);
    if (g.local < 0 || g.local * ATT_TQ >= g.len) return;
    const long long q0 = seg_at(a.q_ptr, g.seg, a.n_seg, a.n_q), q1 = seg_at(a.q_ptr, g.seg + 1, a.n_seg, a.n_q);
    const int n_sub = q1 > q0 ? (int)((q1 - q0 + 31) >> 5) : 0, items = n_sub * rep;
    const int per = (items + a.splits - 1) / a.splits, i0 = min(split * per, items), i1 = min(i0 + per, items);
    const long long qbase = (q0 >> 5) + g.seg, head0 = (long long)kvh * rep;
    const int ki = g.local * ATT_TQ + 32 * w + j, nsk = (g.len + 31) >> 5, wsub = min(g.local * 4 + w, nsk - 1);
    const long long kplace = (g.first >> 5) + g.seg + wsub, ksub = (long long)kvh * a.ns_k + kplace;

constexpr int PIECES = SUB * 2 / 1024;
    const int lz = lane_zero(), tl = tr_lane(lane), even = rot_lane(lane, 0), odd = rot_lane(lane, 1);
    int rep_at = i0 < i1 ? i0 / n_sub : 0, sub_at = i0 < i1 ? i0 % n_sub : 0;            // of the item that is requested next
    Staged<2 * PIECES> st;
    float sr = 0.f;
    int sp = 0;
    u32x4 listed{}, listed_next{};
    Record<KIND, 2> r, rn;
    auto request = [&]() {
        const long long s = (head0 + rep_at) * a.ns_q + qbase + sub_at;
        st.request(w, lane, [&](int c) {
            const int image = c / PIECES;
            return (const char*)(image == 0 ? a.q_r : a.g_r) + s * (SUB * 2) + (c % PIECES) * 1024;
        });
        if (t < 96) sr = a.rows[s * 96 + t];
        if (AXES > 0 && t < AXES * 32) sp = a.qpos[(qbase + sub_at) * (AXES * 32) + t];
        if constexpr (BIAS == LISTED) listed_next = a.by_key[(kplace * a.ns_q + qbase + sub_at) * 64 + lane];
        rn.request(a.rec_q + s + lz);
    };
    auto arrive = [&](int b) {
        st.write_rotated(buf[b], w, lane);
        if (t < 96) rbuf[b][t] = sr;
        if (AXES > 0 && t < AXES * 32) pbuf[b][t] = sp;
        listed = listed_next;
        r = rn;
        r.settle();
    };
    if (i0 < i1) request();

    u32x4 kf[PL][NC], vf[PL][NC];
    {
        const u32x4 *kp = (const u32x4*)(a.k_r + ksub * SUB) + lane, *vp = (const u32x4*)(a.v_r + ksub * SUB) + lane;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int c = 0; c < NC; ++c) { kf[p][c] = kp[(p * NC + c) * 64]; vf[p][c] = vp[(p * NC + c) * 64]; }
    }
    const i32x4 rk = a.rec_k[ksub];
    int ek = 0, ev = 0;                                       // exponents of this key and its value
    if constexpr (KIND != AT_BF16) { ek = block_exp(rk[0]) + a.fix_k[ksub * 32 + j]; ev = block_exp(rk[1]) + a.fix_v[ksub * 32 + j]; }
    int kx = 0, ky = 0, kz = 0;
    float most = 0.f;
    if constexpr (BIAS > 0) {
        if constexpr (AXES > 0) {
            const int* p = a.kpos + kplace * (AXES * 32) + j;
            kx = p[0];
            if (AXES > 1) ky = p[32];
            if (AXES > 2) kz = p[64];
        }
        most = (float)(a.reach * a.reach) + 0.5f;
        if (i0 < i1) fill_biases<BIAS>(lutb, a, (int)head0 + rep_at, t);
    }
    // Exponents of this key's sums, dV of P and dK of dS: as for a query's (attn_dq_kernel).  P is small for every query where a key
    // has little weight, and dS holds <g, o>, the values of all the other keys: neither is bounded by this key's own block.
    int unit_p = UNIT_LEAST, unit_s = UNIT_LEAST;

    f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) { dk[b] = zero16(); dv[b] = zero16(); }
    if (i0 < i1) arrive(0);
    __syncthreads();
    for (int item = i0; item < i1; ++item) {
        const int b = (item - i0) & 1;
        bool next_head = false;
        const long long qsub_at = (head0 + rep_at) * a.ns_q + qbase + sub_at;      // of this item
        if (item + 1 < i1) {
            if (++sub_at == n_sub) { sub_at = 0; ++rep_at; next_head = true; }
        }
        request();
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const u32x4 q1 = rot_read<NC>(buf[b], even, odd, 0, c), g1 = rot_read<NC>(buf[b] + SUB, even, odd, 0, c);
            if constexpr (PL == 2) {
                s = mma<KIND>(rot_read<NC>(buf[b], even, odd, 1, c), kf[0][c], s);
                dp = mma<KIND>(rot_read<NC>(buf[b] + SUB, even, odd, 1, c), vf[0][c], dp);
                s = mma<KIND>(q1, kf[PL - 1][c], s);
                dp = mma<KIND>(g1, vf[PL - 1][c], dp);
            }
            s = mma<KIND>(q1, kf[0][c], s);
            dp = mma<KIND>(g1, vf[0][c], dp);
        }
        const float c = KIND == AT_BF16 ? a.c0 : score_factor(ldexpf(a.c0, block_exp(r.v[0]) + ek));
        const float up = KIND == AT_BF16 ? 1.f : wsub & 1 ? -unit_factor(block_exp(r.v[1]) + ev) : unit_factor(block_exp(r.v[1]) + ev);
        if (KIND != AT_BF16 && block_apart(r.v[0] | r.v[1])) {
            apply_fix(s, row_fix(a.fix_q + qsub_at * 32, h));
            apply_fix(dp, row_fix(a.fix_g + qsub_at * 32, h));
        }
        f32x16 p;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float* rr = rbuf[b] + 8 * q + 4 * h;
            const f32x4 m = *(const f32x4*)rr, norm = *(const f32x4*)(rr + 32), delta = *(const f32x4*)(rr + 64);
            float add[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (BIAS > 0) {
                i32x4 x, y, z;
                if constexpr (AXES > 0) places4<AXES>(pbuf[b] + 8 * q + 4 * h, x, y, z);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int at;
                    if constexpr (AXES > 0) at = place<AXES>(x[e], y[e], z[e], kx, ky, kz, a.reach, most);
                    else at = listed[q] >> (8 * e) & (ATT_MAX_BUCKETS - 1);
                    add[e] = lutb[at];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = 4 * q + e;
                const float x = BIAS > 0 ? __builtin_fmaf(s[n], c, add[e]) - m[e] : __builtin_fmaf(s[n], c, -m[e]);
                float pe = __builtin_amdgcn_exp2f(x);
                if constexpr (KIND != AT_F32) pe *= norm[e];
                const float d = KIND == AT_BF16 ? dp[n] - delta[e] : __builtin_fmaf(dp[n], up, -delta[e]);
                s[n] = pe * d;
                p[n] = pe;
            }
        }
        if constexpr (KIND != AT_BF16) {
            if (block_apart(r.v[0] | r.v[1])) {
                apply_fix(s, row_fix(a.fix_q + qsub_at * 32, h));
                apply_fix(p, row_fix(a.fix_g + qsub_at * 32, h));
            }
            const float most_p = largest16(p), most_s = largest16(s);
            const int eq = block_exp(r.v[0]), eg = block_exp(r.v[1]);
            float fp = ldexpf(1.f, eg - unit_p), fs = ldexpf(1.f, eq - unit_s);
            if (__any(max(eg - unit_p, eq - unit_s) > FACTOR_MOST || fmaxf(most_p * fp, most_s * fs) > UNIT_OVER)) {      // the two halves of a key's queries only meet here
                const int to_p = raised_unit(unit_p, fmaxf(most_p, __shfl_xor(most_p, 32)), eg);
                const int to_s = raised_unit(unit_s, fmaxf(most_s, __shfl_xor(most_s, 32)), eq);
                const float by_p = unit_factor(unit_p - to_p), by_s = unit_factor(unit_s - to_s);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    scale16<DP == 128>(dv[n], by_p);
                    scale16<DP == 128>(dk[n], by_s);
                }
                unit_p = to_p; unit_s = to_s;
                fp = ldexpf(1.f, eg - unit_p); fs = ldexpf(1.f, eq - unit_s);
            }
#pragma unroll
            for (int n = 0; n < 16; ++n) { p[n] *= fp; s[n] *= fs; }
        }
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            float v[8];
            u32x4 phi, plo, shi, slo;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = p[8 * kc + e];
            pack8<KIND>(v, phi, plo);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = s[8 * kc + e];
            pack8<KIND>(v, shi, slo);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const u32x4 g1 = tr_read<DP>(buf[b] + SUB, tl, 0, kc, n), q1 = tr_read<DP>(buf[b], tl, 0, kc, n);
                if constexpr (PL == 2) {
                    dv[n] = mma<KIND>(tr_read<DP>(buf[b] + SUB, tl, 1, kc, n), phi, dv[n]);
                    dk[n] = mma<KIND>(tr_read<DP>(buf[b], tl, 1, kc, n), shi, dk[n]);
                    dv[n] = mma<KIND>(g1, plo, dv[n]);
                    dk[n] = mma<KIND>(q1, slo, dk[n]);
                }
                dv[n] = mma<KIND>(g1, phi, dv[n]);
                dk[n] = mma<KIND>(q1, shi, dk[n]);
            }
        }
        arrive(b ^ 1);
        __syncthreads();
        if (BIAS > 0 && next_head) {                           // the next item is of another head
            fill_biases<BIAS>(lutb, a, (int)head0 + rep_at, t);
            __syncthreads();
        }
    }
    if (ki >= g.len) return;
    const bool keep = (unsigned)rk[2] >> j & 1;                // a masked key has no gradient
    const long long row = g.first + ki;
    float* part = a.part + ((long long)split * 2 * a.kv_heads * a.ns_k + ksub) * 32 * DP + j * DP;
    const long long vpart = (long long)a.kv_heads * a.ns_k * 32 * DP;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * n + 8 * q + 4 * h;
            if (d >= a.dim) continue;
            f32x4 vk, vv;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = dk[n][4 * q + e] * a.scale, y = dv[n][4 * q + e];
                vk[e] = !keep ? 0.f : KIND == AT_BF16 ? x : ldexpf(x, unit_s);
                vv[e] = !keep ? 0.f : KIND == AT_BF16 ? y : ldexpf(y, unit_p);
            }
            if (a.splits > 1) {
                *(f32x4*)(part + d) = vk; *(f32x4*)(part + vpart + d) = vv;
            } else {
                store4<KIND>(a.dk, (row * a.kv_heads + kvh) * a.dim + d, vk);
                store4<KIND>(a.dv, (row * a.kv_heads + kvh) * a.dim + d, vv);
            }
        }
}

// dQ of a query, dK and dV of a key = sum over the splits, in order; one thread per four values.  Memory bound.
template <int KIND>
__global__ __launch_bounds__(256) void attn_dq_sum_kernel(AttnBwd a, int dp) {
    const int quads = a.dim / 4;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x, units = (long long)a.heads * a.ns_q;
    if (item >= units * 32 * quads) return;
    const int quad = (int)(item % quads), i = (int)(item / quads % 32);
    const long long unit = item / quads / 32;
    const int head = (int)(unit / a.ns_q), sub = (int)(unit % a.ns_q);
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, 5, sub);
    if (g.local < 0 || g.local * 32 + i >= g.len) return;
    const float* p = a.q_part + (unit * 32 + i) * dp + 4 * quad;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.q_splits; ++s) v += *(const f32x4*)(p + (long long)s * units * 32 * dp);
    store4<KIND>(a.dq, ((g.first + g.local * 32 + i) * a.heads + head) * a.dim + 4 * quad, v);
}
template <int KIND>
__global__ __launch_bounds__(256) void attn_dkv_sum_kernel(AttnBwd a, int dp) {
    const int quads = a.dim / 4;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x, units = (long long)a.kv_heads * a.ns_k;
    if (item >= units * 32 * quads) return;
    const int quad = (int)(item % quads), i = (int)(item / quads % 32);
    const long long unit = item / quads / 32;
    const int kvh = (int)(unit / a.ns_k), sub = (int)(unit % a.ns_k);
    const Seg g = find_tile(a.k_ptr, a.n_seg, a.n_k, 5, sub);
    if (g.local < 0 || g.local * 32 + i >= g.len) return;
    const float* p = a.part + (unit * 32 + i) * dp + 4 * quad;
    f32x4 k = {0.f, 0.f, 0.f, 0.f}, v = k;
    for (int s = 0; s < a.splits; ++s) {
        k += *(const f32x4*)(p + (long long)(2 * s) * units * 32 * dp);
        v += *(const f32x4*)(p + (long long)(2 * s + 1) * units * 32 * dp);
    }
    const long long at = ((g.first + g.local * 32 + i) * a.kv_heads + kvh) * a.dim + 4 * quad;
    store4<KIND>(a.dk, at, k);
    store4<KIND>(a.dv, at, v);
}

// ------------------------------------------------------------------------------------------------ host
struct BwdSpace { size_t q_r, g_r, k_r, v_r, rec_q, rec_k, fix_q, fix_g, fix_k, fix_v, rows, qpos, kpos, tpart, part, q_part, by_query, by_key, total; int ns_q, ns_k, q_tiles, k_tiles, splits, q_splits; bool listed; };

BwdSpace bwd_space(const MgnAttn& a, bool table_grad) {
    BwdSpace s{};
    const int dp = attn_dp(a.dim), pl = a.dtype == MGN_F32 ? 2 : 1;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t p = at; at += (bytes + 255) & ~(size_t)255; return p; };
    s.ns_q = attn_subtiles(a.n_q, a.n_seg); s.ns_k = attn_subtiles(a.n_k, a.n_seg);
    s.q_tiles = (int)(a.n_q / ATT_TQ) + a.n_seg; s.k_tiles = (int)(a.n_k / ATT_TQ) + a.n_seg;
    // workgroups of the key side: two per compute unit, in shares of at least four query subtiles (backward pass in us for 512 / 768 /
    // 1024 workgroups: 20 000 x 2501, 4 heads of 32, fp32, plane 455 / 446 / 464; 16 segments of 1123 x 804, 8 heads over 2 of 64,
    // bf16 198 / 227 / 211; four of 1339 x 1339, 8 heads of 64, fp16, line 165 / 175 / 174; with 256 the first took 15 % longer)
    const int64_t blocks = attn_tiles(a.n_k, a.n_seg, ATT_TQ) * a.kv_heads, items = (a.n_q / 32 / a.n_seg + 1) * (a.heads / a.kv_heads);
    int64_t sp = blocks > 0 ? 512 / blocks : 1;
    if (sp > items / 4) sp = items / 4;
    s.splits = (int)(sp < 1 ? 1 : sp > 64 ? 64 : sp);
    s.q_splits = attn_round_splits(attn_tiles(a.n_q, a.n_seg, ATT_TQ) * a.heads, a.n_k / a.n_seg, 1);
    const size_t qi = (size_t)a.heads * s.ns_q * pl * 64 * dp, ki = (size_t)a.kv_heads * s.ns_k * pl * 64 * dp;
    s.q_r = take(qi); s.g_r = take(qi); s.k_r = take(ki); s.v_r = take(ki);
    s.rec_q = take((size_t)a.heads * s.ns_q * 16); s.rec_k = take((size_t)a.kv_heads * s.ns_k * 16);
    const size_t row = a.dtype == MGN_BF16 ? 0 : 128, qf = (size_t)a.heads * s.ns_q * row, kf = (size_t)a.kv_heads * s.ns_k * row;
    s.fix_q = take(qf); s.fix_g = take(qf); s.fix_k = take(kf); s.fix_v = take(kf);
    s.rows = take((size_t)a.heads * s.ns_q * 96 * 4);
    // Buckets listed once where a place is dear (a lattice), at least two heads share it and there are subtiles enough to pay for the
    // launch, up to 1 GB in all.  Backward pass in us without and with: 20 000 x 2501, 4 heads of 32, fp32, plane 599 / 510, in space
    // 529 / 463, 16 heads over 2 of 64, bf16, 1642 / 1372, 2 heads of 64, fp32, 445 / 426; 4000 x 1000 114 / 101; 2000 x 500 96 / 99.
    const int64_t tiles = (int64_t)s.ns_q * s.ns_k;
    s.listed = a.bias_table && a.axes > 1 && a.heads > 1 && tiles >= 2048 && tiles <= 1 << 19;
    if (s.listed) { s.by_query = take((size_t)tiles * 1024); s.by_key = take((size_t)tiles * 1024); }
    if (a.bias_table) { s.qpos = take((size_t)s.ns_q * a.axes * 128); s.kpos = take((size_t)s.ns_k * a.axes * 128); }
    if (table_grad) s.tpart = take((size_t)s.q_tiles * s.q_splits * a.heads * a.n_bucket * 8);
    if (s.q_splits > 1) s.q_part = take((size_t)s.q_splits * a.heads * s.ns_q * 32 * dp * 4);
    if (s.splits > 1) s.part = take((size_t)s.splits * 2 * a.kv_heads * s.ns_k * 32 * dp * 4);
    s.total = at;
    return s;
}

// Whether the kernel fits the 160 KB of LDS with this much dynamic memory, which beyond 64 KB has to be asked for.  A launch
// that does not fit is never made: it would end the process's queue, not return an error.  The function's limit is set once for each
// device, to all that is left beside its static memory: it belongs to the function, not to a call, and two threads may be launching.
template <auto kernel>
bool lds_fits(int dynamic) {
    static std::atomic<int> room[64];                          // by device: bytes left, plus one
    if (dynamic == 0) return true;
    int dev;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
    int left = room[dev].load(std::memory_order_acquire) - 1;
    if (left < 0) {
        hipFuncAttributes at;
        if (hipFuncGetAttributes(&at, (const void*)kernel) != hipSuccess || at.sharedSizeBytes > 160 * 1024) return false;
        left = 160 * 1024 - (int)at.sharedSizeBytes;
        if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, left) != hipSuccess) return false;
        room[dev].store(left + 1, std::memory_order_release);
    }
    return dynamic <= left;
}

template <int KIND, int DP, int BIAS>
bool bwd_launch(const AttnBwd& b, const BwdSpace& s, hipStream_t st) {
    const int hist = BIAS > 0 ? (b.tpart ? b.n_bucket * 1024 : 0) + entries<BIAS>(b.reach) * (int)sizeof(Entry) : 0;
    if (!lds_fits<attn_dq_kernel<KIND, DP, BIAS>>(hist)) return false;
    hipLaunchKernelGGL((attn_dq_kernel<KIND, DP, BIAS>), dim3((unsigned)(s.q_tiles * b.heads), (unsigned)s.q_splits), dim3(256), hist, st, b);
    if (b.n_k > 0) hipLaunchKernelGGL((attn_dkv_kernel<KIND, DP, BIAS>), dim3((unsigned)(s.k_tiles * b.kv_heads), (unsigned)s.splits), dim3(256), 0, st, b);
    return true;
}
template <int KIND, int DP>
bool bwd_bias(const AttnBwd& b, const BwdSpace& s, int bias, hipStream_t st) {
    if (s.listed) return bwd_launch<KIND, DP, LISTED>(b, s, st);
    if (bias == 0) return bwd_launch<KIND, DP, 0>(b, s, st);
    if (bias == 1) return bwd_launch<KIND, DP, 1>(b, s, st);
    if (bias == 2) return bwd_launch<KIND, DP, 2>(b, s, st);
    return bwd_launch<KIND, DP, 3>(b, s, st);
}
template <int KIND>
bool bwd_kind(const AttnBwd& b, const BwdSpace& s, int dp, int bias, hipStream_t st) {
    const bool fits = dp == 32 ? bwd_bias<KIND, 32>(b, s, bias, st) : dp == 64 ? bwd_bias<KIND, 64>(b, s, bias, st) : bwd_bias<KIND, 128>(b, s, bias, st);
    if (!fits) return false;
    if (s.q_splits > 1) {
        const long long items = (long long)b.heads * s.ns_q * 32 * (b.dim / 4);
        hipLaunchKernelGGL((attn_dq_sum_kernel<KIND>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, b, dp);
    }
    if (s.splits > 1) {
        const long long items = (long long)b.kv_heads * s.ns_k * 32 * (b.dim / 4);
        hipLaunchKernelGGL((attn_dkv_sum_kernel<KIND>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, b, dp);
    }
    return true;
}

}  // namespace

extern "C" int64_t mgn_attn_bwd_workspace_bytes(const MgnAttn* a, int32_t table_grad) {
    if (attn_check(a, "mgn_attn_bwd_workspace_bytes", true) != 0) return -1;
    return (int64_t)bwd_space(*a, table_grad && a->bias_table).total;
}

extern "C" int mgn_attn_bwd(const MgnAttn* ap, const void* g, int64_t g_st, int64_t g_sh, const void* out, int64_t out_st,
                            int64_t out_sh, const float* stats, void* dq, void* dk, void* dv, float* dtable, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    if (const int rc = attn_check(ap, "mgn_attn_bwd", true)) return rc;
    const MgnAttn& a = *ap;
    const char* bad = nullptr;
    const BwdSpace s = bwd_space(a, dtable != nullptr);
    if (a.n_q > 0 && (!g || !out || !stats || !dq)) bad = "null operand";
    else if (a.n_k > 0 && (!dk || !dv)) bad = "null key or value gradient";
    else if (dtable && !a.bias_table) bad = "a table gradient without a table";
    else if (a.n_q > 0 && (attn_bad_rows(g, g_st, g_sh, a.dtype) || attn_bad_rows(out, out_st, out_sh, a.out_f32 ? MGN_F32 : a.dtype))) bad = "rows must start on 16-byte borders";
    else if (((uintptr_t)dq & 15) || ((uintptr_t)dk & 15) || ((uintptr_t)dv & 15)) bad = "gradients must start on 16-byte borders";
    else if (!workspace || workspace_bytes < (int64_t)s.total) bad = "the workspace is missing or too small";
    if (bad) { mgn_set_error("mgn_attn_bwd: %s", bad); return MGN_E_ARG; }
    char* ws = (char*)workspace;
    const int kind = attn_kind(a.dtype), dp = attn_dp(a.dim), bias = attn_bias(a);
    const hipStream_t st = (hipStream_t)stream;
    auto half = [&](size_t at) { return (unsigned short*)(ws + at); };
    auto ints = [&](size_t at) { return (int*)(ws + at); };
    int *rec_q = (int*)(ws + s.rec_q), *rec_k = (int*)(ws + s.rec_k);
    ImageArgs im{};
    im.n_seg = a.n_seg; im.dim = a.dim;
    int units = 0;
    auto add = [&](const void* x, long long xst, long long xsh, bool query) -> ImageJob& {
        ImageJob& jb = im.job[im.n_job++];
        jb.x = x; jb.st = xst; jb.sh = xsh; jb.ptr = query ? a.q_ptr : a.k_ptr; jb.T = query ? a.n_q : a.n_k;
        jb.heads = query ? a.heads : a.kv_heads; jb.n_sub = query ? s.ns_q : s.ns_k; jb.axes = a.axes;
        jb.first_unit = units; units += jb.heads * jb.n_sub;
        if (!query) jb.mask = a.key_mask;
        return jb;
    };
    if (a.n_q > 0) {
        ImageJob& q = add(a.q, a.q_st, a.q_sh, true);
        q.R = half(s.q_r); q.ex = rec_q; q.fix = ints(s.fix_q); q.pos = bias ? a.q_pos : nullptr; q.pos_out = (int*)(ws + s.qpos);
        ImageJob& o = add(g, g_st, g_sh, true);
        o.R = half(s.g_r); o.ex = rec_q + 1; o.fix = ints(s.fix_g); o.o = out; o.o_f32 = a.out_f32 || a.dtype == MGN_F32; o.o_st = out_st; o.o_sh = out_sh; o.stats = stats; o.rows = (float*)(ws + s.rows);
    }
    if (a.n_k > 0) {
        ImageJob& k = add(a.k, a.k_st, a.k_sh, false);
        k.R = half(s.k_r); k.ex = rec_k; k.fix = ints(s.fix_k); k.valid = rec_k + 2; k.pos = bias ? a.k_pos : nullptr; k.pos_out = (int*)(ws + s.kpos);
        ImageJob& v = add(a.v, a.v_st, a.v_sh, false);
        v.R = half(s.v_r); v.ex = rec_k + 1; v.fix = ints(s.fix_v); v.alternate = kind != AT_BF16;
    }
    im.units = units;
    if (units > 0) mgn_attn_launch_images(kind, dp, &im, stream);
    AttnBwd b{};
    b.q_ptr = a.q_ptr; b.k_ptr = a.k_ptr; b.n_q = a.n_q; b.n_k = a.n_k; b.n_seg = a.n_seg; b.heads = a.heads; b.kv_heads = a.kv_heads; b.dim = a.dim;
    b.c0 = std::min(a.scale * LOG2E, F32_MOST); b.scale = a.scale;
    b.fix_q = ints(s.fix_q); b.fix_g = ints(s.fix_g); b.fix_k = ints(s.fix_k); b.fix_v = ints(s.fix_v);
    b.q_r = half(s.q_r); b.g_r = half(s.g_r); b.k_r = half(s.k_r); b.v_r = half(s.v_r);
    b.rec_q = (const i32x4*)rec_q; b.rec_k = (const i32x4*)rec_k; b.rows = (const float*)(ws + s.rows); b.ns_q = s.ns_q; b.ns_k = s.ns_k;
    b.qpos = (const int*)(ws + s.qpos); b.kpos = (const int*)(ws + s.kpos);
    b.table = a.bias_table; b.lut = a.bucket_lut; b.n_bucket = a.n_bucket; b.reach = a.reach; b.axes = a.axes;
    b.dq = dq; b.dk = dk; b.dv = dv; b.dtable = dtable; b.tpart = dtable ? (double*)(ws + s.tpart) : nullptr; b.q_tiles = s.q_tiles;
    b.zero = a.zero_outside && a.q_ptr; b.splits = s.splits; b.part = (float*)(ws + s.part);
    b.q_splits = s.q_splits; b.q_part = (float*)(ws + s.q_part);
    if (s.listed) {
        b.by_query = (u32x4*)(ws + s.by_query); b.by_key = (u32x4*)(ws + s.by_key);
        if (a.n_q > 0 && a.n_k > 0) {
            const dim3 grid((unsigned)((s.ns_q + 3) / 4), (unsigned)std::min<int64_t>(64, std::max<int64_t>(1, 4096 / ((s.ns_q + 3) / 4))));
            if (a.axes == 2) hipLaunchKernelGGL(attn_buckets_kernel<2>, grid, dim3(256), 0, st, b);
            else hipLaunchKernelGGL(attn_buckets_kernel<3>, grid, dim3(256), 0, st, b);
        }
    }
    const bool fits = kind == AT_BF16 ? bwd_kind<AT_BF16>(b, s, dp, bias, st) : kind == AT_F16 ? bwd_kind<AT_F16>(b, s, dp, bias, st)
                                                                                           : bwd_kind<AT_F32>(b, s, dp, bias, st);
    if (!fits) { mgn_set_error("mgn_attn_bwd: %d buckets at width %d do not fit the compute unit's local memory", a.n_bucket, a.dim); return MGN_E_ARG; }
    if (dtable) hipLaunchKernelGGL(attn_table_kernel, dim3((unsigned)(a.heads * a.n_bucket)), dim3(64), 0, st, b.tpart, dtable, s.q_tiles * s.q_splits, a.heads * a.n_bucket);
    return check_launch("mgn_attn_bwd");
}
