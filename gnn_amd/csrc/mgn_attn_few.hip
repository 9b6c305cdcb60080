// Attention with few queries per segment (a probe point, one step of a stream): keys and values are read once, where they
// lie, in whole rows, and all arithmetic is fp32.
//
// Memory bound: bytes = keys x (key + value row).  A workgroup takes one query token, up to eight query heads that share a
// key head, and one piece of the keys; LPR lanes share a row (8 elements each), so a load of a wave covers 64 / LPR rows; four
// loads (two for fp32) of keys and of values are worked on while as many are on their way.  Every row group keeps its own
// running maximum and sum, joined over the wave by exchanges and over the waves through LDS; pieces are joined in a fixed order.
// Measured: one query in each of 64 streams over 358 608 ragged keys, 16 heads over 4 key heads of 128, bf16, 177 us, 4.2 TB/s
// (a copy reaches 4.8, a plain read 4.0); one query over 100 000 keys, 4 heads of 32, fp32, with bias, 30 us, 3.4 TB/s, of which
// the launches of its two kernels are 8.
#include "mgn_attn_host.h"

#include <type_traits>

namespace {

// Sum over the LPR lanes that share a row, by data-parallel exchanges within groups of 16 lanes (no LDS): neighbours, pairs,
// then mirrored halves -- at each step both partners add the same two numbers, so all lanes hold the same sum.
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
    auto add = [&](auto ctrl) { v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true)); };
    add(std::integral_constant<int, 0xB1>());                        // lanes 1 0 3 2
    add(std::integral_constant<int, 0x4E>());                        // lanes 2 3 0 1
    if constexpr (LPR >= 8) add(std::integral_constant<int, 0x141>());    // mirrored in 8
    if constexpr (LPR >= 16) add(std::integral_constant<int, 0x140>());   // mirrored in 16
    return v;
}

template <int KIND, int LPR, int REP, bool bias>
__global__ __launch_bounds__(256, REP == 8 && (bias || KIND == AT_F32) ? 1 : 2) void attn_few_kernel(AttnFwd a) {
    constexpr int RPW = 64 / LPR, U = KIND == AT_F32 || REP == 8 || (bias && REP == 4) ? 2 : 4;
    __shared__ float joined[4][REP][LPR * 8 + 2];
    __shared__ unsigned char lutb[bias ? 2 * ATT_MAX_REACH + 1 : 1];
    __shared__ float tab[REP][bias ? ATT_MAX_BUCKETS : 1];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, part = lane % LPR, rg = lane / LPR;
    const int rep = a.heads / a.kv_heads, chunks = (rep + REP - 1) / REP;
    const int chunk = blockIdx.x % chunks, kvh = blockIdx.x / chunks % a.kv_heads, split = blockIdx.y;
    const long long row = blockIdx.x / chunks / a.kv_heads;
    int lo = 0, hi = a.n_seg;                                   // the last segment that starts at or before this token
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seg_at(a.q_ptr, mid, a.n_seg, a.n_q) <= row) lo = mid; else hi = mid;
    }
    if (row < seg_at(a.q_ptr, lo, a.n_seg, a.n_q) || row >= seg_at(a.q_ptr, lo + 1, a.n_seg, a.n_q)) {
        const int quads = a.dim / 4;
        if (a.zero && split == 0)
            for (int x = t; x < REP * quads; x += 256)
                if (chunk * REP + x / quads < rep)
                    store4<KIND>(a.out, row * a.o_st + (kvh * rep + chunk * REP + x / quads) * a.o_sh + 4 * (x % quads), f32x4{0.f, 0.f, 0.f, 0.f});
        return;
    }
    const long long f = seg_at(a.k_ptr, lo, a.n_seg, a.n_k), e = seg_at(a.k_ptr, lo + 1, a.n_seg, a.n_k);
    const long long len = e > f ? e - f : 0, per = (len + a.splits - 1) / a.splits;
    const long long k0 = f + (split * per < len ? split * per : len), k1 = k0 + per < f + len ? k0 + per : f + len;

    const int head0 = kvh * rep + chunk * REP, d = 8 * part;
    float q[REP][8], o[REP][8], m[REP], l[REP];
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        const bool on = chunk * REP + r < rep && d < a.dim;
        if (on) load8<KIND>(a.q, row * a.q_st + (head0 + r) * a.q_sh + d, q[r]);
#pragma unroll
        for (int c = 0; c < 8; ++c) { q[r][c] = on ? q[r][c] * a.c0 : 0.f; o[r][c] = 0.f; }
        m[r] = -__builtin_inff(); l[r] = 0.f;
    }
    struct Piece { Raw8<KIND> k[U], v[U]; int use, x[bias ? U : 1], y[bias ? U : 1], z[bias ? U : 1]; } one, two;
    auto request = [&](Piece& p, long long base) {
        p.use = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long key = base + (u * 4 + w) * RPW + rg;
            const bool use = key < k1 && (!a.mask || a.mask[key]);
            p.use |= use ? 1 << u : 0;
            p.k[u].zero(); p.v[u].zero();
            if (use && d < a.dim) {
                p.k[u].load(a.k, key * a.k_st + kvh * a.k_sh + d);
                p.v[u].load(a.v, key * a.v_st + kvh * a.v_sh + d);
            }
            if constexpr (bias) {
                p.x[u] = p.y[u] = p.z[u] = 0;
                const int* at = a.k_pos + key * a.axes;
                if (use) p.x[u] = at[0];
                if (use && a.axes > 1) p.y[u] = at[1];
                if (use && a.axes > 2) p.z[u] = at[2];
            }
        }
    };
    request(one, k0);                                           // on its way while the bias is set up
    int qx = 0, qy = 0, qz = 0;
    const float most = (float)(a.reach * a.reach) + 0.5f;
    if (bias) {
        const int* p = a.q_pos + row * a.axes;
        qx = p[0];
        if (a.axes > 1) qy = p[1];
        if (a.axes > 2) qz = p[2];
        const int entries = a.axes == 1 ? 2 * a.reach + 1 : a.reach + 1;
        for (int r = t; r < entries; r += 256) lutb[r] = (unsigned char)min(max(a.lut[r], 0), a.n_bucket - 1);
        for (int r = t; r < REP * a.n_bucket; r += 256) {
            const int hd = r / a.n_bucket, b = r % a.n_bucket;
            tab[hd][b] = chunk * REP + hd < rep ? bias_log2(a.table[(head0 + hd) * a.n_bucket + b]) : 0.f;
        }
        __syncthreads();
    }
    auto take = [&](const Piece& p) {
        float s[U][REP];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float kv[8];
            p.k[u].get(kv);
            int bucket = 0;
            if constexpr (bias)
                bucket = lutb[a.axes == 1 ? place<1>(qx, qy, qz, p.x[u], p.y[u], p.z[u], a.reach, most)
                                          : place<3>(qx, qy, qz, p.x[u], p.y[u], p.z[u], a.reach, most)];   // an axis that is not there is zero on both sides
#pragma unroll
            for (int r = 0; r < REP; ++r) {
                float x = 0.f;
#pragma unroll
                for (int c = 0; c < 8; ++c) x = __builtin_fmaf(q[r][c], kv[c], x);
                x = row_sum<LPR>(x);
                if constexpr (bias) x += tab[r][bucket];
                s[u][r] = p.use >> u & 1 ? x : -__builtin_inff();
            }
        }
#pragma unroll
        for (int r = 0; r < REP; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, s[u][r]);
            const float to = top == -__builtin_inff() ? 0.f : top, al = __builtin_amdgcn_exp2f(m[r] - to);
            m[r] = top;
            l[r] *= al;
#pragma unroll
            for (int c = 0; c < 8; ++c) o[r][c] *= al;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - to);
                l[r] += s[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float vv[8];
            p.v[u].get(vv);
#pragma unroll
            for (int r = 0; r < REP; ++r)
#pragma unroll
                for (int c = 0; c < 8; ++c) o[r][c] = __builtin_fmaf(s[u][r], vv[c], o[r][c]);
        }
    };
    // two sets of rows that swap roles: the next one is on its way while this one is worked on
    constexpr int STEP = 4 * RPW * U;
    for (long long base = k0; base < k1; base += 2 * STEP) {
        request(two, base + STEP);
        take(one);
        request(one, base + 2 * STEP);
        if (base + STEP < k1) take(two);
    }
    // join the row groups of the wave, then the four waves
#pragma unroll
    for (int r = 0; r < REP; ++r) {
#pragma unroll
        for (int x = LPR; x < 64; x <<= 1) {
            const float m2 = __shfl_xor(m[r], x), l2 = __shfl_xor(l[r], x), top = fmaxf(m[r], m2), to = top == -__builtin_inff() ? 0.f : top;
            const float f1 = __builtin_amdgcn_exp2f(m[r] - to), f2 = __builtin_amdgcn_exp2f(m2 - to);
            // the lower lane's share is added first on both sides: both hold the same sums
            const bool low = (lane & x) == 0;
            const float a1 = l[r] * f1, a2 = l2 * f2;
            l[r] = low ? a1 + a2 : a2 + a1;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float o2 = __shfl_xor(o[r][c], x) * f2, o1 = o[r][c] * f1;
                o[r][c] = low ? o1 + o2 : o2 + o1;
            }
            m[r] = top;
        }
        if (rg == 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) joined[w][r][part * 8 + c] = o[r][c];
            if (part == 0) { joined[w][r][LPR * 8] = m[r]; joined[w][r][LPR * 8 + 1] = l[r]; }
        }
    }
    __syncthreads();
    const int dp = attn_dp_device(a.dim);
    for (int x = t; x < REP * LPR * 2; x += 256) {              // four output values each
        const int r = x / (LPR * 2), c = 4 * (x % (LPR * 2));
        if (chunk * REP + r >= rep || c >= a.dim) continue;
        float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) top = fmaxf(top, joined[g][r][LPR * 8]);
        const float to = top == -__builtin_inff() ? 0.f : top;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float s = __builtin_amdgcn_exp2f(joined[g][r][LPR * 8] - to);
            sum += s * joined[g][r][LPR * 8 + 1];
#pragma unroll
            for (int n = 0; n < 4; ++n) v[n] += s * joined[g][r][c + n];
        }
        const int head = head0 + r;
        if (a.splits > 1) {
            const long long at = ((long long)split * a.heads + head) * a.n_q + row;
            *(f32x4*)(a.part + at * dp + c) = v;
            if (c == 0) { a.part_ml[2 * at] = top; a.part_ml[2 * at + 1] = sum; }
        } else {
            v *= inverse_sum(sum);
            store4<KIND>(a.out, row * a.o_st + head * a.o_sh + c, v);
            if (KIND != AT_F32 && a.out32) *(f32x4*)(a.out32 + (row * a.heads + head) * a.dim + c) = v;
            if (c == 0 && a.stats) {
                a.stats[(long long)head * a.n_q + row] = top;
                a.stats[(long long)(a.heads + head) * a.n_q + row] = sum;
            }
        }
    }
}

template <int KIND, int LPR, int REP>
void few_bias(const AttnFwd& f, dim3 grid, hipStream_t st) {
    if (f.table) hipLaunchKernelGGL((attn_few_kernel<KIND, LPR, REP, true>), grid, dim3(256), 0, st, f);
    else hipLaunchKernelGGL((attn_few_kernel<KIND, LPR, REP, false>), grid, dim3(256), 0, st, f);
}
template <int KIND, int LPR>
void few_rep(const AttnFwd& f, int rep, dim3 grid, hipStream_t st) {
    if (rep == 1) few_bias<KIND, LPR, 1>(f, grid, st);
    else if (rep == 2) few_bias<KIND, LPR, 2>(f, grid, st);
    else if (rep == 4) few_bias<KIND, LPR, 4>(f, grid, st);
    else few_bias<KIND, LPR, 8>(f, grid, st);
}
template <int KIND>
void few_kind(const AttnFwd& f, int rep, dim3 grid, hipStream_t st) {
    if (f.dim <= 32) few_rep<KIND, 4>(f, rep, grid, st);
    else if (f.dim <= 64) few_rep<KIND, 8>(f, rep, grid, st);
    else few_rep<KIND, 16>(f, rep, grid, st);
}

}  // namespace

int mgn_attn_launch_few(int kind, const AttnFwd* fp, void* stream) {
    const AttnFwd& f = *fp;
    MgnAttn a{};
    a.heads = f.heads; a.kv_heads = f.kv_heads; a.n_q = f.n_q;
    const int rep = attn_few_chunk(a);
    const dim3 grid((unsigned)attn_few_blocks(a), (unsigned)f.splits);
    const hipStream_t st = (hipStream_t)stream;
    if (kind == AT_BF16) few_kind<AT_BF16>(f, rep, grid, st);
    else if (kind == AT_F16) few_kind<AT_F16>(f, rep, grid, st);
    else few_kind<AT_F32>(f, rep, grid, st);
    return 0;
}
