// Attention of one set of states over another, forwards: operand images, the tiled kernel, the join of split key ranges.
#include "mgn_attn.h"
#include "mgn_attn_host.h"

namespace {

// ---------------------------------------------------------------------------------------------- operand images
// One wave per (head, subtile): lane (i, h) reads the elements 16 c + 8 h .. + 7 of token i, which are its share of image R;
// image T is read back from a row-major copy in LDS.  Memory bound: 4 bytes read and 4 (R) or 8 (R and T) written per element.
// Measured: the four images of a backward pass over 17 973 queries, 8 heads of 64, and 12 870 keys, 2 heads, bf16: 24 us for
// 105 MB, 4.4 TB/s.
template <int KIND, int DP>
__global__ __launch_bounds__(256) void attn_image_kernel(ImageArgs a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, LD = DP + 2;
    __shared__ unsigned short tr[4][32 * LD];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const int unit = min((int)blockIdx.x * 4 + w, a.units - 1);          // the last units are done twice, with equal results
    int jb = 0;
    while (jb + 1 < a.n_job && unit >= a.job[jb + 1].first_unit) ++jb;
    const ImageJob& job = a.job[jb];
    const int u = unit - job.first_unit, head = u % job.heads, sub = u / job.heads;
    const Seg g = find_tile(job.ptr, a.n_seg, job.T, 5, sub);
    const int tok = 32 * g.local + i;
    const bool inside = g.local >= 0 && tok < g.len;
    const long long row = inside ? g.first + tok : 0;
    const bool use = inside && (!job.mask || job.mask[row]);

    float v[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * h;
        if (use && d < a.dim) load8<KIND>(job.x, row * job.st + head * job.sh + d, v[c]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
    const long long at = (long long)head * job.n_sub + sub;
    if (job.rows) {
        float m = 0.f, l = 0.f, dot = 0.f;
        if (use) {
            m = job.stats[(long long)head * job.T + row];
            l = job.stats[(long long)(job.heads + head) * job.T + row];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 16 * c + 8 * h;
                if (d < a.dim) {
                    float o[8];
                    const long long at = row * job.o_st + head * job.o_sh + d;
                    if (job.o_f32) load8<AT_F32>(job.o, at, o); else load8<KIND>(job.o, at, o);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(v[c][e], o[e], dot);
                }
            }
        }
        dot += __shfl_xor(dot, 32);
        const float il = inverse_sum(l);
        if constexpr (KIND == AT_F32) {
            dot *= il;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] *= il;
        }
        if (h == 0) {
            float* r = job.rows + at * 96;
            r[i] = zero_bits(l) ? __builtin_inff() : m;       // an empty row, or none: every exp2(score - m) is zero
            r[32 + i] = KIND == AT_F32 ? 1.f : il;
            r[64 + i] = zero_bits(l) ? 0.f : dot;
        }
    }
    if (job.pos && head == 0 && h == 0)
        for (int ax = 0; ax < job.axes; ++ax) job.pos_out[((long long)sub * job.axes + ax) * 32 + i] = inside ? job.pos[row * job.axes + ax] : 0;

    int ex = 0;
    bool apart = false;
    if constexpr (KIND != AT_BF16) {
        const float top = row_top<NC>(v), most = wave_max(top);
        ex = scale_exp<KIND>(most);
        int er = ex;
        apart = __any(top > 0.f && top < most * (1.f / (1 << APART)));
        if (apart && top > 0.f && top < most * (1.f / (1 << APART))) er = scale_exp<KIND>(top);
        const float by = job.alternate && (g.local & 1) ? -pow2i(-er) : pow2i(-er);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] *= by;
        if (h == 0) job.fix[at * 32 + i] = er - ex;
    }
    const unsigned long long bits = __ballot(use);
    if (lane == 0) {
        job.ex[at * 4] = block_word(ex, apart);
        if (job.valid) job.valid[at * 4] = (int)(unsigned)bits;
    }
    u32x4 hi[NC], lo[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) pack8<KIND>(v[c], hi[c], lo[c]);
    if (job.R) {
        u32x4* dst = (u32x4*)(job.R + at * (PL * 32 * DP)) + lane;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            dst[c * 64] = hi[c];
            if constexpr (PL == 2) dst[(NC + c) * 64] = lo[c];
        }
    }
    if (!a.transposed) return;
    // every wave of the workgroup takes both rounds, whatever its job asks for: the barriers are met by all
#pragma unroll
    for (int p = 0; p < PL; ++p) {
        __syncthreads();
        unsigned* line = (unsigned*)(tr[w] + i * LD);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) line[8 * c + 4 * h + e] = p ? lo[c][e] : hi[c][e];
        __syncthreads();
        if (job.Tt) {
            u32x4* dst = (u32x4*)(job.Tt + at * (PL * 32 * DP)) + lane;
#pragma unroll
            for (int kc = 0; kc < 2; ++kc)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    const unsigned short* src = tr[w] + (16 * kc + 4 * h) * LD + 32 * b + i;
                    u32x4 r;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t0 = e < 2 ? 2 * e : 8 + 2 * (e - 2);
                        r[e] = (unsigned)src[t0 * LD] | ((unsigned)src[(t0 + 1) * LD] << 16);
                    }
                    dst[((p * 2 + kc) * (DP / 32) + b) * 64] = r;
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------- tiled kernel
// A workgroup: 128 queries of one head, 32 per wave, against the key range of its split, 32 keys at a time.  Both products
// are transposed (S^T = K Q^T, O^T = V^T P^T), so a lane holds scores of ONE query: the running maximum and sum of its softmax
// are a register each, and its probabilities are the second product's operand as they stand.
// P2: 16-bit types with probabilities in two planes, for the fp32 outputs that the gradient of a bias table needs.
//
// The two or three waves of a SIMD fall into step at the barriers, so a wave overlaps its matrix and vector work itself: the
// scores of step t + 1 are on the matrix unit between the exponentials of step t, and step t's sums between the bias and the
// maximum of step t + 1 (the sched_group_barriers deal the instructions out).  Keys are therefore staged one step further
// ahead than values.  The maximum is only raised when a score exceeds it by more than OVER (base 2): until then probabilities up
// to 2^OVER are as good as ones up to 1, and rescaling the sums, due in most steps of a wave otherwise, becomes rare.
//
// Measured, images included: 8192 x 8192, 8 heads of 128, bf16, 277 us, 0.99 PFLOP/s, 78 % of a large library product:
// bound by the matrix unit and by what exponentials do not hide under it.  20 000 x 2501, 4 heads of 32, fp32, places on a plane:
// 172 us with the join of two pieces; bound by the vector unit (340 vector instructions a step beside 12 products).
template <int KIND, int DP, int BIAS, bool P2, int NW>
__global__ __launch_bounds__(64 * NW, (KIND == AT_F32 && DP == 128) || NW == 8 ? 1 : 2) void attn_fwd_kernel(AttnFwd a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, NB = DP / 32, SUB = PL * 32 * DP;
    constexpr int SHIFT = KIND == AT_BF16 ? 0 : 15 - OVER;     // probabilities are scaled up: small ones keep their bits in fp16
    constexpr int PIECES = SUB * 2 / 1024;                     // of 1 KB
    __shared__ __attribute__((aligned(1024))) unsigned short kbuf[2][SUB];
    __shared__ __attribute__((aligned(1024))) unsigned short vbuf[2][SUB];
    __shared__ __attribute__((aligned(16))) int pbuf[BIAS ? 2 : 1][BIAS ? 128 : 1];
    __shared__ float lutb[BIAS == 1 ? 2 * ATT_MAX_REACH + 1 : BIAS ? ATT_MAX_REACH + 1 : 1];

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.heads, kvh = head / (a.heads / a.kv_heads), split = blockIdx.y;
    if (a.zero) zero_outside<KIND>(a.q_ptr, a.n_seg, a.n_q, a.out, a.o_st, a.o_sh, a.heads, a.dim);
    constexpr int TILE_LOG = NW == 8 ? 8 : 7;
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, TILE_LOG, blockIdx.x / a.heads);
    if (g.local < 0 || (g.local << TILE_LOG) >= g.len) return;
    const long long k0 = seg_at(a.k_ptr, g.seg, a.n_seg, a.n_k), k1 = seg_at(a.k_ptr, g.seg + 1, a.n_seg, a.n_k);
    const int n_sub = k1 > k0 ? (int)((k1 - k0 + 31) >> 5) : 0;
    const int per = (n_sub + a.splits - 1) / a.splits;
    const int s0 = min(split * per, n_sub), n_it = min(s0 + per, n_sub) - s0, last = n_it - 1;
    const long long sub0 = (k0 >> 5) + g.seg + s0;             // first subtile of the range in the images
    const char* kimg = (const char*)(a.kimg + ((long long)kvh * a.ns_k + sub0) * SUB);
    const char* vimg = (const char*)(a.vimg + ((long long)kvh * a.ns_k + sub0) * SUB);
    const i32x4* rec = a.rec + (long long)kvh * a.ns_k + sub0;
    const int *kfix = a.kfix + ((long long)kvh * a.ns_k + sub0) * 32, *vfix = a.vfix + ((long long)kvh * a.ns_k + sub0) * 32;

    Staged<PIECES, NW> sk, sv;
    int sp = 0;
    auto request_k = [&](int it) {                             // keys and, with a bias, their places
        sk.request(w, lane, [&](int c) { return kimg + (long long)it * (SUB * 2) + c * 1024; });
        if (BIAS > 0 && t < a.axes * 32) sp = a.kpos[(sub0 + it) * a.axes * 32 + t];
    };
    auto request_v = [&](int it) { sv.request(w, lane, [&](int c) { return vimg + (long long)it * (SUB * 2) + c * 1024; }); };
    auto arrive_k = [&](int b) {
        sk.write(kbuf[b], w, lane);
        if (BIAS > 0 && t < a.axes * 32) pbuf[b][t] = sp;
    };
    if (n_it > 0) { request_k(0); request_v(0); }

    const int qi = (g.local << TILE_LOG) + 32 * w + j;
    const long long row = g.first + min(qi, g.len - 1);
    u32x4 qh[NC], ql[NC];                                       // the queries' operand, scaled per row
    int eq = 0;                                                 // by 2^-eq
    {
        float v[NC][8], top = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 16 * c + 8 * h;
            if (d < a.dim) load8<KIND>(a.q, row * a.q_st + head * a.q_sh + d, v[c]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
            if constexpr (KIND != AT_BF16)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[c][e]));
        }
        if constexpr (KIND != AT_BF16) {
            eq = scale_exp<KIND>(fmaxf(top, __shfl_xor(top, 32)));
            const float by = pow2i(-eq);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] *= by;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) pack8<KIND>(v[c], qh[c], ql[c]);
    }
    int qx = 0, qy = 0, qz = 0;
    float most = 0.f;
    if constexpr (BIAS > 0) {
        const int* p = a.q_pos + row * a.axes;
        qx = p[0];
        if (BIAS > 1) qy = p[1];
        if (BIAS > 2) qz = p[2];
        most = (float)(a.reach * a.reach) + 0.5f;
        const int entries = BIAS == 1 ? 2 * a.reach + 1 : a.reach + 1;
        for (int r = t; r < entries; r += 64 * NW)
            lutb[r] = bias_log2(a.table[head * a.n_bucket + min(max(a.lut[r], 0), a.n_bucket - 1)]);
    }
    f32x16 o[NB], s;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = zero16();
    float m = -__builtin_inff(), l = 0.f, c = 0.f, unit = SUM_UNIT_LEAST;
    u32x4 kf[PL][NC], vf[PL][2][NB];
    auto key_operands = [&](int b) {
        const u32x4* kp = (const u32x4*)kbuf[b] + lane;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int x = 0; x < NC; ++x) kf[p][x] = kp[(p * NC + x) * 64];
    };
    auto scores = [&]() {
        f32x16 x = zero16();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if constexpr (PL == 2) {
                x = mma<KIND>(kf[PL - 1][n], qh[n], x);
                x = mma<KIND>(kf[0][n], ql[n], x);
            }
            x = mma<KIND>(kf[0][n], qh[n], x);
        }
        return x;
    };
    auto biased = [&](f32x16& x, int b) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            i32x4 px, py, pz;
            places4<BIAS>(pbuf[b] + 8 * q + 4 * h, px, py, pz);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[4 * q + e] = __builtin_fmaf(x[4 * q + e], c, lutb[place<BIAS>(qx, qy, qz, px[e], py[e], pz[e], a.reach, most)]);
        }
    };
    // scores of a step: scaled (with a bias; without one when the exponentials are taken), masked; returns the largest
    auto finish = [&](f32x16& x, int b, int word, int valid, int it) {
        const bool apart = KIND != AT_BF16 && block_apart(word);
        c = KIND == AT_BF16 ? a.c0 : score_factor(ldexpf(a.c0, eq + block_exp(word)));
        if constexpr (BIAS > 0) biased(x, b);
        if (valid != -1 || apart) {
            if (apart) {                                        // key rows with exponents of their own
                if constexpr (BIAS > 0) x = scores();           // the keys' operand is still there: once more, without the bias
                apply_fix(x, row_fix(kfix + (long long)it * 32, h));
                int again = b;
                if constexpr (BIAS == 1) asm volatile("" : "+s"(again));        // a line's places are cheap: found anew (kept for this
                if constexpr (BIAS > 0) biased(x, again);                       // branch, 8192 x 4096, 8 heads of 32, 183 instead of 175 us)
            }
            mask_scores(x, valid, h);
        }
        float top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) top = fmaxf(top, fmaxf(x[e], x[e + 1]));
        if constexpr (BIAS == 0) top *= c;                      // c > 0
        return top;                                             // of this lane's half of the keys
    };
    Record<KIND> r, rn, rnn;                                    // exponents and mask of steps t, t + 1, t + 2
    const int lz = lane_zero();
    float top = -__builtin_inff();
    if (n_it > 0) {
        r.request(rec + lz);
        rn.request(rec + min(1, last) + lz);
        r.settle(); rn.settle();
        arrive_k(0);
        sv.write(vbuf[0], w, lane);
        request_k(min(1, last));
        __syncthreads();
        key_operands(0);
        s = scores();
        top = finish(s, 0, r.v[0], r.v[2], 0);
        arrive_k(1);
        __syncthreads();
    }
    for (int it = 0; it < n_it; ++it) {
        const int b = it & 1;
        request_v(min(it + 1, last));
        request_k(min(it + 2, last));
        rnn.request(rec + min(it + 2, last) + lz);              // on its way like the operands: nothing waits for it here
        key_operands(b ^ 1);
        const u32x4* vp = (const u32x4*)vbuf[b] + lane;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int kc = 0; kc < 2; ++kc)
#pragma unroll
                for (int n = 0; n < NB; ++n) vf[p][kc][n] = vp[((p * 2 + kc) * NB + n) * 64];
        const float ev = (float)block_exp(r.v[1]);              // the values' exponent
        const bool apart = KIND != AT_BF16 && block_apart(r.v[1]);
        if (__any((KIND == AT_BF16 ? top - m : top - m + fmaxf(ev - unit, 0.f)) > (float)OVER) || apart) {
            const float most = fmaxf(top, __shfl_xor(top, 32)), lowered = raise_max(m, l, most);       // the two halves of a
            const float zero = m == -__builtin_inff() ? 0.f : m;                                       // query's keys only meet here
            float need = most - zero, by;
            if (apart) {                                        // every value row has its own exponent: its probability takes it
                const RowFix f = row_fix(vfix + (long long)it * 32, h);
                need = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = (BIAS > 0 ? s[e] : s[e] * c) - zero;
                    l += __builtin_amdgcn_exp2f(s[e]);
                    s[e] += (float)f.f[e >> 2][e & 3];
                    need = fmaxf(need, s[e]);
                }
                need = fmaxf(need, __shfl_xor(need, 32));
            }
            if constexpr (KIND == AT_BF16) by = __builtin_amdgcn_exp2f(lowered);
            else by = raise_unit(unit, lowered, need + ev);
#pragma unroll
            for (int n = 0; n < NB; ++n) scale16<KIND == AT_F32 && DP == 128>(o[n], by);
        }
        float base = m == -__builtin_inff() || apart ? 0.f : m;
        if (BIAS > 0 && __any(fabsf(base) > 0x1p20f)) {         // biases near the ends of their type: a shift added to the
#pragma unroll                                                  // maximum would be rounded away
            for (int e = 0; e < 16; ++e) s[e] -= base;
            base = 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- scores of the next step on the matrix unit, exponentials of this one on the vector unit
        const float sh = KIND == AT_BF16 ? 0.f : (float)SHIFT + fmaxf(ev - unit, (float)FAR_EXP), back = sh - base, cs = apart ? 1.f : c;
        f32x16 sn = scores();
        float sum = 0.f;
        u32x4 ph[2], plo[2];
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pv[e] = __builtin_amdgcn_exp2f(BIAS > 0 ? s[8 * kc + e] + back : __builtin_fmaf(s[8 * kc + e], cs, back));
                sum += pv[e];
            }
            pack8<KIND, P2 || PL == 2>(pv, ph[kc], plo[kc]);
        }
        constexpr int VALU1 = PL == 2 || P2 ? 96 : 56, MFMA1 = NC * (PL == 2 ? 3 : 1);
#pragma unroll
        for (int n = 0; n < MFMA1; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VALU1 / MFMA1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- sums of this step on the matrix unit, bias and maximum of the next one on the vector unit
        l += KIND == AT_BF16 ? sum : sum * (apart ? 0.f : __builtin_amdgcn_exp2f(-sh));
#pragma unroll
        for (int kc = 0; kc < 2; ++kc)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                if constexpr (PL == 2) o[n] = mma<KIND>(vf[PL - 1][kc][n], ph[kc], o[n]);
                if constexpr (P2 || PL == 2) o[n] = mma<KIND>(vf[0][kc][n], plo[kc], o[n]);
                o[n] = mma<KIND>(vf[0][kc][n], ph[kc], o[n]);
            }
        s = sn;
        r = rn;
        top = finish(s, b ^ 1, r.v[0], r.v[2], min(it + 1, last));
        sv.write(vbuf[b ^ 1], w, lane);
        arrive_k(b);
        rn = rnn;
        rn.settle();
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    if (qi >= g.len) return;
    const float inv = a.splits > 1 ? 1.f : inverse_sum(l);
    const long long prow = ((long long)split * a.heads + head) * a.n_q + row;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * n + 8 * q + 4 * h;
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = KIND == AT_BF16 ? o[n][4 * q + e] * inv : scale_real(o[n][4 * q + e] * inv, unit - SHIFT);
            if (a.splits > 1) *(f32x4*)(a.part + prow * DP + d) = v;
            else if (d < a.dim) {
                store4<KIND>(a.out, row * a.o_st + head * a.o_sh + d, v);
                if (P2) *(f32x4*)(a.out32 + (row * a.heads + head) * a.dim + d) = v;
            }
        }
    if (h == 0) {
        if (a.splits > 1) {
            a.part_ml[2 * prow] = m; a.part_ml[2 * prow + 1] = l;
        } else if (a.stats) {
            a.stats[(long long)head * a.n_q + row] = m;
            a.stats[(long long)(a.heads + head) * a.n_q + row] = l;
        }
    }
}

// ---------------------------------------------------------------------------------------------- tiled kernel, two heads
// The tiled kernel with a bias by distance on a lattice where a wave takes two heads of the same 32 queries: the place of a
// (query, key) pair, a dozen vector instructions, is found once for both, and the products of the second head are issued before
// the exponentials of the first.  Bound by the vector unit.  Measured: 100 000 queries x 1225 keys, 4 heads of 32, places on a
// plane, 364 us in fp32 and 243 us in fp16 (a head at a time 382 and 298).
constexpr int HEADS = 2;
template <int KIND, int DP, int BIAS, bool P2>
__global__ __launch_bounds__(256, DP == 32 && KIND != AT_F32 ? 3 : 2) void attn_fwd_heads_kernel(AttnFwd a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, NB = DP / 32, SUB = PL * 32 * DP;
    constexpr int SHIFT = KIND == AT_BF16 ? 0 : 15 - OVER, PIECES = SUB * 2 / 1024;
    constexpr int LUTS = ATT_MAX_REACH + 4;
    __shared__ __attribute__((aligned(1024))) unsigned short buf[2][HEADS * 2 * SUB];         // [head][keys, values]
    __shared__ __attribute__((aligned(16))) int pbuf[2][128];
    __shared__ float lutb[HEADS * LUTS];

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const int groups = a.heads / HEADS, head0 = blockIdx.x % groups * HEADS, rep = a.heads / a.kv_heads, split = blockIdx.y;
    if (a.zero) zero_outside<KIND>(a.q_ptr, a.n_seg, a.n_q, a.out, a.o_st, a.o_sh, a.heads, a.dim);
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, 7, blockIdx.x / groups);
    if (g.local < 0 || g.local * ATT_TQ >= g.len) return;
    const long long k0 = seg_at(a.k_ptr, g.seg, a.n_seg, a.n_k), k1 = seg_at(a.k_ptr, g.seg + 1, a.n_seg, a.n_k);
    const int n_sub = k1 > k0 ? (int)((k1 - k0 + 31) >> 5) : 0;
    const int per = (n_sub + a.splits - 1) / a.splits;
    const int s0 = min(split * per, n_sub), n_it = min(s0 + per, n_sub) - s0, last = n_it - 1;
    const long long sub0 = (k0 >> 5) + g.seg + s0;

    Staged<HEADS * 2 * PIECES> st;
    int sp = 0;
    auto request = [&](int it) {
        st.request(w, lane, [&](int c) {
            const int image = c / PIECES;
            const long long at = ((long long)((head0 + image / 2) / rep) * a.ns_k + sub0 + it) * (SUB * 2) + (c % PIECES) * 1024;
            return (const char*)(image & 1 ? a.vimg : a.kimg) + at;
        });
        if (t < a.axes * 32) sp = a.kpos[(sub0 + it) * a.axes * 32 + t];
    };
    auto arrive = [&](int b) {
        st.write(buf[b], w, lane);
        if (t < a.axes * 32) pbuf[b][t] = sp;
    };
    if (n_it > 0) request(0);

    const int qi = g.local * ATT_TQ + 32 * w + j;
    const long long row = g.first + min(qi, g.len - 1);
    u32x4 qh[HEADS][NC], ql[PL == 2 ? HEADS : 1][NC];
    int eq[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        float v[NC][8], top = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 16 * c + 8 * h;
            if (d < a.dim) load8<KIND>(a.q, row * a.q_st + (head0 + i) * a.q_sh + d, v[c]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
            if constexpr (KIND != AT_BF16)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[c][e]));
        }
        eq[i] = 0;
        if constexpr (KIND != AT_BF16) {
            eq[i] = scale_exp<KIND>(fmaxf(top, __shfl_xor(top, 32)));
            const float by = pow2i(-eq[i]);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] *= by;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) pack8<KIND>(v[c], qh[i][c], ql[PL == 2 ? i : 0][c]);
    }
    const int* qp = a.q_pos + row * a.axes;
    const int qx = qp[0], qy = qp[1], qz = BIAS > 2 ? qp[2] : 0;
    const float most = (float)(a.reach * a.reach) + 0.5f;
    for (int r = t; r <= a.reach; r += 256) {
        const int b = min(max(a.lut[r], 0), a.n_bucket - 1);
#pragma unroll
        for (int i = 0; i < HEADS; ++i) lutb[i * LUTS + r] = bias_log2(a.table[(head0 + i) * a.n_bucket + b]);
    }
    const i32x4* rec[HEADS];
    const int lz = lane_zero();
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        rec[i] = a.rec + (long long)((head0 + i) / rep) * a.ns_k + sub0;
    }
    f32x16 o[HEADS][NB];
    float m[HEADS], l[HEADS], unit[HEADS];
    Record<KIND> r[HEADS], rn[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        m[i] = -__builtin_inff(); l[i] = 0.f; unit[i] = SUM_UNIT_LEAST;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[i][b] = zero16();
        if (n_it > 0) { r[i].request(rec[i] + lz); r[i].settle(); }
    }
    if (n_it > 0) arrive(0);
    __syncthreads();
    for (int it = 0; it < n_it; ++it) {
        const int b = it & 1;
        request(min(it + 1, last));
#pragma unroll
        for (int i = 0; i < HEADS; ++i) rn[i].request(rec[i] + min(it + 1, last) + lz);
        auto scores = [&](int i) {
            const u32x4* kp = (const u32x4*)(buf[b] + i * 2 * SUB) + lane;
            f32x16 s = zero16();
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (PL == 2) {
                    s = mma<KIND>(kp[(NC + c) * 64], qh[i][c], s);
                    s = mma<KIND>(kp[c * 64], ql[i][c], s);
                }
                s = mma<KIND>(kp[c * 64], qh[i][c], s);
            }
            return s;
        };
        f32x16 s = scores(0);
        int idx[16];                                            // byte offsets into the biases by place
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            i32x4 x, y, z;
            places4<BIAS>(pbuf[b] + 8 * q + 4 * h, x, y, z);
#pragma unroll
            for (int e = 0; e < 4; ++e) idx[4 * q + e] = 4 * place<BIAS>(qx, qy, qz, x[e], y[e], z[e], a.reach, most);
        }
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            const float c = KIND == AT_BF16 ? a.c0 : score_factor(ldexpf(a.c0, eq[i] + block_exp(r[i].v[0])));
            const long long block = ((long long)((head0 + i) / rep) * a.ns_k + sub0 + it) * 32;
            auto biased = [&] {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(s[e], c, *(const float*)((const char*)(lutb + i * LUTS) + idx[e]));
            };
            biased();
            const bool apart_k = KIND != AT_BF16 && block_apart(r[i].v[0]);
            if (r[i].v[2] != -1 || apart_k) {
                if (apart_k) {                                  // key rows with exponents of their own: once more, without the bias
                    s = scores(i);
                    apply_fix(s, row_fix(a.kfix + block, h));
                    biased();
                }
                mask_scores(s, r[i].v[2], h);
            }
            float top = fmaxf(s[0], s[1]);
#pragma unroll
            for (int e = 2; e < 16; e += 2) top = fmaxf(top, fmaxf(s[e], s[e + 1]));
            const float ev = (float)block_exp(r[i].v[1]);       // the values' exponent
            const bool apart = KIND != AT_BF16 && block_apart(r[i].v[1]);
            if (__any((KIND == AT_BF16 ? top - m[i] : top - m[i] + fmaxf(ev - unit[i], 0.f)) > (float)OVER) || apart) {   // as in attn_fwd_kernel
                const float most = fmaxf(top, __shfl_xor(top, 32)), lowered = raise_max(m[i], l[i], most);
                const float zero = m[i] == -__builtin_inff() ? 0.f : m[i];
                float need = most - zero, by;
                if (apart) {
                    const RowFix f = row_fix(a.vfix + block, h);
                    need = -__builtin_inff();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[e] -= zero;
                        l[i] += __builtin_amdgcn_exp2f(s[e]);
                        s[e] += (float)f.f[e >> 2][e & 3];
                        need = fmaxf(need, s[e]);
                    }
                    need = fmaxf(need, __shfl_xor(need, 32));
                }
                if constexpr (KIND == AT_BF16) by = __builtin_amdgcn_exp2f(lowered);
                else by = raise_unit(unit[i], lowered, need + ev);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[i][n][e] *= by;
            }
            float base = m[i] == -__builtin_inff() || apart ? 0.f : m[i];
            if (__any(fabsf(base) > 0x1p20f)) {                 // biases near the ends of their type (see attn_fwd_kernel)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] -= base;
                base = 0.f;
            }
            f32x16 next;
            if (i + 1 < HEADS) next = scores(i + 1);
            const float sh = KIND == AT_BF16 ? 0.f : (float)SHIFT + fmaxf(ev - unit[i], (float)FAR_EXP), back = sh - base;
            const u32x4* vp = (const u32x4*)(buf[b] + (i * 2 + 1) * SUB) + lane;
            float sum = 0.f;
#pragma unroll
            for (int kc = 0; kc < 2; ++kc) {
                float pv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pv[e] = __builtin_amdgcn_exp2f(s[8 * kc + e] + back);
                    sum += pv[e];
                }
                u32x4 ph, plo;
                pack8<KIND, P2 || PL == 2>(pv, ph, plo);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if constexpr (PL == 2) o[i][n] = mma<KIND>(vp[((2 + kc) * NB + n) * 64], ph, o[i][n]);
                    if constexpr (P2 || PL == 2) o[i][n] = mma<KIND>(vp[(kc * NB + n) * 64], plo, o[i][n]);
                    o[i][n] = mma<KIND>(vp[(kc * NB + n) * 64], ph, o[i][n]);
                }
            }
            l[i] += KIND == AT_BF16 ? sum : sum * (apart ? 0.f : __builtin_amdgcn_exp2f(-sh));
            s = next;
        }
        arrive(b ^ 1);
#pragma unroll
        for (int i = 0; i < HEADS; ++i) { r[i] = rn[i]; r[i].settle(); }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        l[i] += __shfl_xor(l[i], 32);
        const int head = head0 + i;
        if (qi >= g.len) continue;
        const float inv = a.splits > 1 ? 1.f : inverse_sum(l[i]);
        const long long prow = ((long long)split * a.heads + head) * a.n_q + row;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * n + 8 * q + 4 * h;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = KIND == AT_BF16 ? o[i][n][4 * q + e] * inv : scale_real(o[i][n][4 * q + e] * inv, unit[i] - SHIFT);
                if (a.splits > 1) *(f32x4*)(a.part + prow * DP + d) = v;
                else if (d < a.dim) {
                    store4<KIND>(a.out, row * a.o_st + head * a.o_sh + d, v);
                    if (P2) *(f32x4*)(a.out32 + (row * a.heads + head) * a.dim + d) = v;
                }
            }
        if (h == 0) {
            if (a.splits > 1) {
                a.part_ml[2 * prow] = m[i]; a.part_ml[2 * prow + 1] = l[i];
            } else if (a.stats) {
                a.stats[(long long)head * a.n_q + row] = m[i];
                a.stats[(long long)(a.heads + head) * a.n_q + row] = l[i];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- small problems
// One launch and no images: a workgroup takes 32 queries of a head, its four waves every fourth subtile of the keys, which they
// read where they lie (keys row by row, values column by column, both straight into operand registers) and scale themselves;
// the waves' sums meet in LDS.  Latency bound: what counts is the length of the chain, not the conversions done again in
// every workgroup.  Measured: 561 x 280, 4 heads of 32, fp32: 10.9 us, 14 to 15 us as a call from Python.
template <int KIND, int DP, int BIAS, bool P2>
__global__ __launch_bounds__(256, DP == 128 || (KIND == AT_F32 && DP == 64) ? 1 : 2) void attn_small_kernel(AttnFwd a) {
    constexpr int PL = planes<KIND>(), NC = DP / 16, NB = DP / 32, LD = DP + 4;
    constexpr int SHIFT = KIND == AT_BF16 ? 0 : 13;
    __shared__ float lutb[BIAS ? 2 * ATT_MAX_REACH + 1 : 1];
    __shared__ __attribute__((aligned(16))) float sums[4][32][LD];
    __shared__ float mls[4][2][32];

    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.heads, kvh = head / (a.heads / a.kv_heads);
    if (a.zero) zero_outside<KIND>(a.q_ptr, a.n_seg, a.n_q, a.out, a.o_st, a.o_sh, a.heads, a.dim);
    const Seg g = find_tile(a.q_ptr, a.n_seg, a.n_q, 5, blockIdx.x / a.heads);
    if (g.local < 0 || g.local * 32 >= g.len) return;
    const long long k0 = seg_at(a.k_ptr, g.seg, a.n_seg, a.n_k), k1 = seg_at(a.k_ptr, g.seg + 1, a.n_seg, a.n_k);
    const int klen = (int)(k1 > k0 ? k1 - k0 : 0), n_sub = (klen + 31) >> 5;
    const int qi = g.local * 32 + j;
    const long long row = g.first + min(qi, g.len - 1);

    u32x4 qh[NC], ql[NC];
    int eq = 0;
    {
        float v[NC][8], top = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 16 * c + 8 * h;
            if (d < a.dim) load8<KIND>(a.q, row * a.q_st + head * a.q_sh + d, v[c]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[c][e]));
        }
        if constexpr (KIND != AT_BF16) {
            eq = scale_exp<KIND>(fmaxf(top, __shfl_xor(top, 32)));
            const float by = pow2i(-eq);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] *= by;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) pack8<KIND>(v[c], qh[c], ql[c]);
    }
    int qx = 0, qy = 0, qz = 0;
    float most = 0.f;
    if constexpr (BIAS > 0) {
        const int* p = a.q_pos + row * a.axes;
        qx = p[0];
        if (BIAS > 1) qy = p[1];
        if (BIAS > 2) qz = p[2];
        most = (float)(a.reach * a.reach) + 0.5f;
        const int entries = BIAS == 1 ? 2 * a.reach + 1 : a.reach + 1;
        for (int r = t; r < entries; r += 256)
            lutb[r] = bias_log2(a.table[head * a.n_bucket + min(max(a.lut[r], 0), a.n_bucket - 1)]);
        __syncthreads();
    }

    f32x16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = zero16();
    float m = -__builtin_inff(), l = 0.f, unit = SUM_UNIT_LEAST;
    for (int sub = w; sub < n_sub; sub += 4) {
        const int key = 32 * sub + j;
        const bool use = key < klen && (!a.mask || a.mask[k0 + key]);
        const unsigned valid = (unsigned)__ballot(use);         // both halves of the wave hold the same keys
        u32x4 kh[NC], kl[NC], vh[2][NB], vl[2][NB];
        int ek = 0, e1 = 0, fk = 0;                             // exponents of the keys and values; what row j's own differs by
        bool apart_k = false, apart_v = false;
        int kx[BIAS ? 16 : 1], ky[BIAS > 1 ? 16 : 1], kz[BIAS > 2 ? 16 : 1];
        auto places = [&] {                                     // of this lane's keys
            if constexpr (BIAS > 0)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int* p = a.k_pos + (k0 + min(32 * sub + 8 * (e >> 2) + 4 * h + (e & 3), klen - 1)) * a.axes;
                    kx[e] = p[0]; ky[BIAS > 1 ? e : 0] = BIAS > 1 ? p[1] : 0; kz[BIAS > 2 ? e : 0] = BIAS > 2 ? p[2] : 0;
                }
        };
        float fv[16];                                           // what the values' rows of this lane's scores have of their own
        {
            if constexpr (DP == 32) places();                   // requested with the rows; wider heads have no registers for them
            float v[NC][8];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 16 * c + 8 * h;
                if (use && d < a.dim) load8<KIND>(a.k, (k0 + key) * a.k_st + kvh * a.k_sh + d, v[c]);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
            }
            float x[2][NB][8];                                  // values: column 32 b + j of keys 16 kc + 4 h + (0 .. 3, 8 .. 11)
#pragma unroll
            for (int kc = 0; kc < 2; ++kc)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int n = 16 * kc + 4 * h + (e & 3) + 8 * (e >> 2), d = 32 * b + j;
                        x[kc][b][e] = (valid >> n & 1) && d < a.dim ? load1<KIND>(a.v, (k0 + 32 * sub + n) * a.v_st + kvh * a.v_sh + d) : 0.f;
                    }
            if constexpr (KIND != AT_BF16) {
                // Sizes of the key rows (a lane has half a row) and of the value rows (a lane has a column: 16 elements of each half's rows)
                float most[16], topk = 0.f, topv = 0.f, low = F32_MOST;
                auto sizes = [&](bool finite) {
                    topk = finite ? finite_top<NC>(v) : topk;
                    topv = 0.f;
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        most[n] = 0.f;
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const float y = fabsf(x[n >> 3][b][n & 7]);
                            most[n] = fmaxf(most[n], finite && !finite_bits(y) ? 0.f : y);
                        }
                        topv = fmaxf(topv, most[n]);
                    }
                };
                float mk, mv;                                   // of the block
                auto meet = [&] {
                    topk = fmaxf(topk, __shfl_xor(topk, 32));
                    mk = topk; mv = fmaxf(topv, __shfl_xor(topv, 32));
#pragma unroll
                    for (int o2 = 16; o2 > 0; o2 >>= 1) { mk = fmaxf(mk, __shfl_xor(mk, o2)); mv = fmaxf(mv, __shfl_xor(mv, o2)); }
                    ek = scale_exp<KIND>(mk); e1 = scale_exp<KIND>(mv);
                };
                constexpr float FAR = 1.f / (1 << APART);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) topk = fmaxf(topk, fabsf(v[c][e]));
                sizes(false);
                meet();
                // None of the value rows is far below the others if in either half of the wave one lane has no small element (masked
                // rows aside).  Where that does not clear them, or there is an infinity, the rows are looked at one by one.
                if (valid == 0xffffffffu)
#pragma unroll
                    for (int n = 0; n < 16; ++n) low = fminf(low, most[n]);
                else
#pragma unroll
                    for (int n = 0; n < 16; ++n) low = valid >> (4 * h) >> (8 * (n >> 2) + (n & 3)) & 1 ? fminf(low, most[n]) : low;
                const unsigned long long clear = __ballot(low >= mv * FAR);
                if ((unsigned)clear == 0 || clear >> 32 == 0 || __any((topk > 0.f && topk < mk * FAR) || !finite_bits(fmaxf(mk, mv)))) {
                    sizes(true);
                    meet();
                    const bool far = topk > 0.f && topk < mk * FAR;
                    apart_k = __any(far);
                    if (far) fk = scale_exp<KIND>(topk) - ek;
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
#pragma unroll
                        for (int o2 = 16; o2 > 0; o2 >>= 1) most[n] = fmaxf(most[n], __shfl_xor(most[n], o2));
                        const int own = most[n] > 0.f && most[n] < mv * FAR ? scale_exp<KIND>(most[n]) : e1;
                        fv[n] = (float)(own - e1);
                        apart_v |= __any(own != e1);
#pragma unroll
                        for (int b = 0; b < NB; ++b) x[n >> 3][b][n & 7] = ldexpf(x[n >> 3][b][n & 7], e1 - own);
                    }
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[c][e] = ldexpf(v[c][e], -fk);
                }
                const float bk = pow2i(-ek), bv = pow2i(-e1);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[c][e] *= bk;
#pragma unroll
                for (int n = 0; n < 16; ++n)
#pragma unroll
                    for (int b = 0; b < NB; ++b) x[n >> 3][b][n & 7] *= bv;
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) pack8<KIND>(v[c], kh[c], kl[c]);
#pragma unroll
            for (int kc = 0; kc < 2; ++kc)
#pragma unroll
                for (int b = 0; b < NB; ++b) pack8<KIND>(x[kc][b], vh[kc][b], vl[kc][b]);
        }
        f32x16 s = zero16();
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if constexpr (PL == 2) {
                s = mma<KIND>(kl[c], qh[c], s);
                s = mma<KIND>(kh[c], ql[c], s);
            }
            s = mma<KIND>(kh[c], qh[c], s);
        }
        const float c = KIND == AT_BF16 ? a.c0 : score_factor(ldexpf(a.c0, eq + ek));
        if (apart_k)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = ldexpf(s[e], __shfl(fk, 8 * (e >> 2) + 4 * h + (e & 3)));
        if constexpr (DP != 32) places();
        float top = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int n = 8 * (e >> 2) + 4 * h + (e & 3);
            float x = s[e] * c;
            if constexpr (BIAS > 0)
                x = __builtin_fmaf(s[e], c, lutb[place<BIAS>(qx, qy, qz, kx[e], ky[BIAS > 1 ? e : 0], kz[BIAS > 2 ? e : 0], a.reach, most)]);
            s[e] = valid >> n & 1 ? x : -__builtin_inff();
            top = fmaxf(top, s[e]);
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float lowered = raise_max(m, l, top), base = m == -__builtin_inff() ? 0.f : m;
        float by, need = top - base;
        if constexpr (KIND == AT_BF16) {
            by = __builtin_amdgcn_exp2f(lowered);
        } else {
            if (apart_v) {
                need = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < 16; ++e) need = fmaxf(need, s[e] - base + fv[e]);
                need = fmaxf(need, __shfl_xor(need, 32));
            }
            by = raise_unit(unit, lowered, need + (float)e1);
        }
        auto shift = [&](float x) { return __builtin_amdgcn_exp2f((float)SHIFT + fminf(fmaxf(x - unit, (float)FAR_EXP), 110.f)); };  // finite: no key yet
        const float sh = KIND == AT_BF16 ? 1.f : shift((float)e1);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] *= by;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] - base);
            l += s[e];
        }
        if constexpr (KIND != AT_BF16) {
            if (apart_v)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= shift((float)e1 + fv[e]);
            else
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= sh;
        }
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            float pv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) pv[e] = s[8 * kc + e];
            u32x4 ph, plo;
            pack8<KIND, P2 || PL == 2>(pv, ph, plo);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                if constexpr (PL == 2) o[n] = mma<KIND>(vl[kc][n], ph, o[n]);
                if constexpr (P2 || PL == 2) o[n] = mma<KIND>(vh[kc][n], plo, o[n]);
                o[n] = mma<KIND>(vh[kc][n], ph, o[n]);
            }
        }
    }
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = KIND == AT_BF16 ? o[n][4 * q + e] : scale_real(o[n][4 * q + e], unit - SHIFT);
            *(f32x4*)&sums[w][j][32 * n + 8 * q + 4 * h] = v;
        }
    if (h == 0) { mls[w][0][j] = m; mls[w][1][j] = l; }
    __syncthreads();
    for (int x = t; x < 32 * (DP / 4); x += 256) {
        const int r = x / (DP / 4), d = 4 * (x % (DP / 4));
        if (g.local * 32 + r >= g.len || d >= a.dim) continue;
        float top = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) top = fmaxf(top, mls[n][0][r]);
        const float base = top == -__builtin_inff() ? 0.f : top;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float f = __builtin_amdgcn_exp2f(mls[n][0][r] - base);
            total = __builtin_fmaf(f, mls[n][1][r], total);
            v += f * *(const f32x4*)&sums[n][r][d];
        }
        v *= inverse_sum(total);
        const long long out = g.first + g.local * 32 + r;
        store4<KIND>(a.out, out * a.o_st + head * a.o_sh + d, v);
        if (P2) *(f32x4*)(a.out32 + (out * a.heads + head) * a.dim + d) = v;
        if (d == 0 && a.stats) {
            a.stats[(long long)head * a.n_q + out] = top;
            a.stats[(long long)(a.heads + head) * a.n_q + out] = total;
        }
    }
}

// ---------------------------------------------------------------------------------------------- join of split key ranges
// o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.  A workgroup per (query, head) -- one wave where there are few pieces --:
// the lanes first hold the factors of the pieces, then share the output's quads, groups of lanes taking every so-manieth piece
// (latency bound: the loads of a group do not depend on each other); fixed order.  Rows that belong to no segment are left.
template <int KIND, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attn_join_kernel(AttnFwd a) {
    constexpr int QUADS = DP / 4, GROUPS = 64 * NW / QUADS;
    __shared__ float fac[ATT_MAX_SPLITS], part_l[NW];
    __shared__ f32x4 sums[NW][QUADS];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int head = blockIdx.x % a.heads;
    const long long row = blockIdx.x / a.heads, stride = a.heads * a.n_q, at = head * a.n_q + row;
    float m = -__builtin_inff();
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * stride + at)]);
    m = wave_max(m);                                             // every wave finds it for itself
    const float base = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f;
    for (int s = t; s < a.splits; s += 64 * NW) {
        const f32x2 ml = *(const f32x2*)(a.part_ml + 2 * (s * stride + at));
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        fac[s] = f;
        l = __builtin_fmaf(f, ml[1], l);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    if (lane == 0) part_l[w] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) l += part_l[x];
    const int quad = t % QUADS, group = t / QUADS;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = group; s < a.splits; s += GROUPS) o += fac[s] * *(const f32x4*)(a.part + (s * stride + at) * DP + 4 * quad);
#pragma unroll
    for (int x = QUADS; x < 64; x <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
    if constexpr (NW > 1) {
        if (lane < QUADS) sums[w][lane] = o;
        __syncthreads();
        if (t < QUADS) {
            o = sums[0][t];
#pragma unroll
            for (int x = 1; x < NW; ++x) o += sums[x][t];
        }
    }
    if (row < seg_at(a.q_ptr, 0, a.n_seg, a.n_q) || row >= seg_at(a.q_ptr, a.n_seg, a.n_seg, a.n_q)) return;
    if (t < QUADS && 4 * quad < a.dim) {
        o *= inverse_sum(l);
        store4<KIND>(a.out, row * a.o_st + head * a.o_sh + 4 * quad, o);
        if (KIND != AT_F32 && a.out32) *(f32x4*)(a.out32 + (row * a.heads + head) * a.dim + 4 * quad) = o;
    }
    if (t == 0 && a.stats) {
        a.stats[(long long)head * a.n_q + row] = m;
        a.stats[(long long)(a.heads + head) * a.n_q + row] = l;
    }
}

// The same for up to eight pieces: four outputs per thread, which reads all factors itself.  Memory bound.  Measured: 20 000
// queries, 4 heads of 32, two pieces, 9.0 us, 3.5 TB/s (a wave per query and head 34 us).
template <int KIND, int DP>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnFwd a) {
    constexpr int QUADS = DP / 4;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x, stride = a.heads * a.n_q;
    const int quad = (int)(item % QUADS), head = (int)(item / QUADS % a.heads);
    const long long row = item / QUADS / a.heads, at = head * a.n_q + row;
    if (row < seg_at(a.q_ptr, 0, a.n_seg, a.n_q) || row >= seg_at(a.q_ptr, a.n_seg, a.n_seg, a.n_q)) return;
    float m = -__builtin_inff(), l = 0.f;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * stride + at)]);
    const float base = m == -__builtin_inff() ? 0.f : m;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const f32x2 ml = *(const f32x2*)(a.part_ml + 2 * (s * stride + at));
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        l = __builtin_fmaf(f, ml[1], l);
        o += f * *(const f32x4*)(a.part + (s * stride + at) * DP + 4 * quad);
    }
    if (4 * quad < a.dim) {
        o *= inverse_sum(l);
        store4<KIND>(a.out, row * a.o_st + head * a.o_sh + 4 * quad, o);
        if (KIND != AT_F32 && a.out32) *(f32x4*)(a.out32 + (row * a.heads + head) * a.dim + 4 * quad) = o;
    }
    if (quad == 0 && a.stats) {
        a.stats[(long long)head * a.n_q + row] = m;
        a.stats[(long long)(a.heads + head) * a.n_q + row] = l;
    }
}

template <int KIND, int DP>
void join_dp(const AttnFwd& f, hipStream_t st) {
    const dim3 grid((unsigned)(f.n_q * f.heads));
    if (f.splits <= 8) hipLaunchKernelGGL((attn_join_rows_kernel<KIND, DP>), dim3((unsigned)((f.n_q * f.heads * (DP / 4) + 255) / 256)), dim3(256), 0, st, f);
    else if (f.splits > 32) hipLaunchKernelGGL((attn_join_kernel<KIND, DP, 4>), grid, dim3(256), 0, st, f);
    else hipLaunchKernelGGL((attn_join_kernel<KIND, DP, 1>), grid, dim3(64), 0, st, f);
}
template <int KIND>
void join_kind(const AttnFwd& f, int dp, hipStream_t st) {
    if (dp == 32) join_dp<KIND, 32>(f, st);
    else if (dp == 64) join_dp<KIND, 64>(f, st);
    else join_dp<KIND, 128>(f, st);
}

template <int KIND, int DP, int BIAS, bool P2>
void fwd_launch(const AttnFwd& f, bool small, dim3 grid, hipStream_t st) {
    if (small) {
        hipLaunchKernelGGL((attn_small_kernel<KIND, DP, BIAS, P2>), grid, dim3(256), 0, st, f);
        return;
    }
    if constexpr (BIAS > 1 && (DP == 32 || (DP == 64 && KIND != AT_F32)))
        if (f.share == HEADS) {
            hipLaunchKernelGGL((attn_fwd_heads_kernel<KIND, DP, BIAS, P2>), grid, dim3(256), 0, st, f);
            return;
        }
    if constexpr (BIAS == 0 && DP == 128 && KIND != AT_F32)
        if (f.waves == 8) {
            hipLaunchKernelGGL((attn_fwd_kernel<KIND, DP, BIAS, P2, 8>), grid, dim3(512), 0, st, f);
            return;
        }
    hipLaunchKernelGGL((attn_fwd_kernel<KIND, DP, BIAS, P2, 4>), grid, dim3(256), 0, st, f);
}
template <int KIND, int DP>
void fwd_bias(const AttnFwd& f, bool small, int bias, dim3 grid, hipStream_t st) {
    constexpr bool TWO = KIND != AT_F32;
    if (f.out32) {
        if (bias == 0) fwd_launch<KIND, DP, 0, TWO>(f, small, grid, st);
        else if (bias == 1) fwd_launch<KIND, DP, 1, TWO>(f, small, grid, st);
        else if (bias == 2) fwd_launch<KIND, DP, 2, TWO>(f, small, grid, st);
        else fwd_launch<KIND, DP, 3, TWO>(f, small, grid, st);
    } else {
        if (bias == 0) fwd_launch<KIND, DP, 0, false>(f, small, grid, st);
        else if (bias == 1) fwd_launch<KIND, DP, 1, false>(f, small, grid, st);
        else if (bias == 2) fwd_launch<KIND, DP, 2, false>(f, small, grid, st);
        else fwd_launch<KIND, DP, 3, false>(f, small, grid, st);
    }
}
template <int KIND>
void fwd_kind(const AttnFwd& f, bool small, int dp, int bias, dim3 grid, hipStream_t st) {
    if (dp == 32) fwd_bias<KIND, 32>(f, small, bias, grid, st);
    else if (dp == 64) fwd_bias<KIND, 64>(f, small, bias, grid, st);
    else fwd_bias<KIND, 128>(f, small, bias, grid, st);
}
template <int KIND>
void image_kind(const ImageArgs& a, int dp, hipStream_t st) {
    const dim3 grid((a.units + 3) / 4);
    if (dp == 32) hipLaunchKernelGGL((attn_image_kernel<KIND, 32>), grid, dim3(256), 0, st, a);
    else if (dp == 64) hipLaunchKernelGGL((attn_image_kernel<KIND, 64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_image_kernel<KIND, 128>), grid, dim3(256), 0, st, a);
}

// workspace of the forward pass, in this order (256-byte aligned pieces)
struct FwdSpace { size_t kimg, vimg, rec, kfix, vfix, kpos, part, ml, total; int ns_k, splits; };

FwdSpace fwd_space(const MgnAttn& a, bool few, bool small) {
    FwdSpace s{};
    const int dp = attn_dp(a.dim), pl = a.dtype == MGN_F32 ? 2 : 1;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t p = at; at += (bytes + 255) & ~(size_t)255; return p; };
    s.ns_k = attn_subtiles(a.n_k, a.n_seg);
    s.splits = few ? attn_few_splits(a) : small ? 1 : attn_fwd_splits(a);
    if (!few && !small) {
        s.kimg = take((size_t)a.kv_heads * s.ns_k * pl * 64 * dp);
        s.vimg = take((size_t)a.kv_heads * s.ns_k * pl * 64 * dp);
        s.rec = take((size_t)a.kv_heads * s.ns_k * 16);
        const size_t fix = a.dtype == MGN_BF16 ? 0 : (size_t)a.kv_heads * s.ns_k * 128;
        s.kfix = take(fix); s.vfix = take(fix);
        s.kpos = take(a.bias_table ? (size_t)(s.ns_k + 1) * a.axes * 128 : 0);
    }
    if (s.splits > 1) {
        s.part = take((size_t)s.splits * a.heads * a.n_q * dp * 4);
        s.ml = take((size_t)s.splits * a.heads * a.n_q * 8);
    }
    s.total = at;
    return s;
}

}  // namespace

int mgn_attn_launch_images(int kind, int dp, const void* args, void* stream) {
    const ImageArgs& a = *(const ImageArgs*)args;
    const hipStream_t st = (hipStream_t)stream;
    if (kind == AT_BF16) image_kind<AT_BF16>(a, dp, st);
    else if (kind == AT_F16) image_kind<AT_F16>(a, dp, st);
    else image_kind<AT_F32>(a, dp, st);
    return 0;
}

extern "C" int64_t mgn_attn_fwd_workspace_bytes(const MgnAttn* a) {
    if (attn_check(a, "mgn_attn_fwd_workspace_bytes", false) != 0) return -1;
    const bool few = attn_is_few(*a);
    return (int64_t)fwd_space(*a, few, !few && attn_is_small(*a)).total;
}

extern "C" int mgn_attn_fwd(const MgnAttn* ap, void* out, int64_t out_st, int64_t out_sh, float* stats, float* out32, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    if (const int rc = attn_check(ap, "mgn_attn_fwd", false)) return rc;
    const MgnAttn& a = *ap;
    if (a.n_q == 0) return 0;
    const bool few = attn_is_few(a), small = !few && attn_is_small(a);
    const FwdSpace sp = fwd_space(a, few, small);
    if (!out || (sp.total > 0 && (!workspace || workspace_bytes < (int64_t)sp.total))) {
        mgn_set_error("mgn_attn_fwd: null output, or a workspace of %lld bytes where %lld are needed", (long long)workspace_bytes, (long long)sp.total);
        return MGN_E_ARG;
    }
    if (attn_bad_rows(out, out_st, out_sh, a.dtype)) { mgn_set_error("mgn_attn_fwd: output rows must be 16-byte aligned"); return MGN_E_ARG; }
    if ((uintptr_t)out32 & 15) { mgn_set_error("mgn_attn_fwd: out32 must start on a 16-byte border"); return MGN_E_ARG; }
    char* ws = (char*)workspace;
    const int kind = attn_kind(a.dtype), dp = attn_dp(a.dim), bias = attn_bias(a);
    const hipStream_t st = (hipStream_t)stream;
    AttnFwd f{};
    f.q = a.q; f.q_st = a.q_st; f.q_sh = a.q_sh;
    f.k = a.k; f.k_st = a.k_st; f.k_sh = a.k_sh; f.v = a.v; f.v_st = a.v_st; f.v_sh = a.v_sh; f.mask = a.key_mask; f.k_pos = a.k_pos;
    f.q_ptr = a.q_ptr; f.k_ptr = a.k_ptr; f.n_seg = a.n_seg; f.n_q = a.n_q; f.n_k = a.n_k;
    f.heads = a.heads; f.kv_heads = a.kv_heads; f.dim = a.dim; f.c0 = std::min(a.scale * LOG2E, F32_MOST);
    f.q_pos = a.q_pos; f.table = a.bias_table; f.lut = a.bucket_lut; f.n_bucket = a.n_bucket; f.reach = a.reach; f.axes = a.axes;
    f.out = out; f.o_st = out_st; f.o_sh = out_sh; f.stats = stats; f.out32 = a.dtype == MGN_F32 ? nullptr : out32; f.splits = sp.splits;
    f.zero = a.zero_outside && a.q_ptr;
    if (sp.splits > 1) { f.part = (float*)(ws + sp.part); f.part_ml = (float*)(ws + sp.ml); }
    if (few) {
        mgn_attn_launch_few(kind, &f, stream);
    } else {
        unsigned short *kimg = (unsigned short*)(ws + sp.kimg), *vimg = (unsigned short*)(ws + sp.vimg);
        int* rec = (int*)(ws + sp.rec);
        int* kpos = (int*)(ws + sp.kpos);
        if (a.n_k > 0 && !small) {
            ImageArgs im{};
            const int units = sp.ns_k * a.kv_heads;
            im.n_job = 2; im.transposed = 1; im.units = 2 * units; im.n_seg = a.n_seg; im.dim = a.dim;
            ImageJob& k = im.job[0];
            k.x = a.k; k.st = a.k_st; k.sh = a.k_sh; k.ptr = a.k_ptr; k.mask = a.key_mask; k.T = a.n_k; k.heads = a.kv_heads; k.n_sub = sp.ns_k;
            k.R = kimg; k.ex = rec; k.fix = (int*)(ws + sp.kfix); k.valid = rec + 2; k.pos = bias ? a.k_pos : nullptr; k.pos_out = kpos; k.axes = a.axes;
            ImageJob& v = im.job[1];
            v = k; v.x = a.v; v.st = a.v_st; v.sh = a.v_sh; v.first_unit = units; v.R = nullptr; v.Tt = vimg; v.ex = rec + 1; v.fix = (int*)(ws + sp.vfix); v.valid = nullptr; v.pos = nullptr;
            mgn_attn_launch_images(kind, dp, &im, stream);
        }
        f.kimg = kimg; f.vimg = vimg; f.rec = (const i32x4*)rec; f.ns_k = sp.ns_k; f.kpos = kpos;
        f.kfix = (const int*)(ws + sp.kfix); f.vfix = (const int*)(ws + sp.vfix);
        f.waves = small ? 4 : attn_fwd_waves(a);
        f.share = small ? 1 : attn_fwd_share(a);
        const dim3 grid((unsigned)((a.n_q / (small ? 32 : 32 * f.waves) + a.n_seg) * (a.heads / f.share)), (unsigned)sp.splits);
        if (kind == AT_BF16) fwd_kind<AT_BF16>(f, small, dp, bias, grid, st);
        else if (kind == AT_F16) fwd_kind<AT_F16>(f, small, dp, bias, grid, st);
        else fwd_kind<AT_F32>(f, small, dp, bias, grid, st);
    }
    if (sp.splits > 1) {
        if (kind == AT_BF16) join_kind<AT_BF16>(f, dp, st);
        else if (kind == AT_F16) join_kind<AT_F16>(f, dp, st);
        else join_kind<AT_F32>(f, dp, st);
    }
    return check_launch("mgn_attn_fwd");
}
