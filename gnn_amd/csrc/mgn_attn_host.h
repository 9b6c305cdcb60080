// Host side of the attention entry points: argument checks, launch shapes, kernel arguments.
#pragma once
#include "mgn_attn.h"

#include <algorithm>
#include <cmath>

// Arguments of the forward kernels (tiled, few queries, join).
struct AttnFwd {
    const void *q, *k, *v; long long q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const uint8_t* mask; const int* k_pos;
    const int *q_ptr, *k_ptr; long long n_q, n_k; int n_seg, heads, kv_heads, dim; float c0;
    const unsigned short *kimg, *vimg; const i32x4* rec; int ns_k; const int *kfix, *vfix, *kpos;
    const int* q_pos; const float* table; const int* lut; int n_bucket, reach, axes;
    void* out; long long o_st, o_sh; float *stats, *out32;
    int splits; float *part, *part_ml;
    int waves, share;                                     // of a workgroup of the tiled kernel; heads that a wave takes
    int zero;                                             // rows outside all segments become zeros
};

int mgn_attn_launch_few(int kind, const AttnFwd* f, void* stream);      // mgn_attn_few.hip

namespace {

inline int attn_kind(int dtype) { return dtype == MGN_BF16 ? AT_BF16 : dtype == MGN_F16 ? AT_F16 : AT_F32; }
inline int attn_dp(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }
inline int attn_bias(const MgnAttn& a) { return a.bias_table ? a.axes : 0; }      // axes of the bias's places; 0: no bias
inline int attn_subtiles(int64_t n, int n_seg) { return (int)(n / 32) + n_seg; }

inline bool attn_bad_rows(const void* p, int64_t st, int64_t sh, int dtype) {
    const int per = dtype == MGN_F32 ? 4 : 8;                           // elements of 16 bytes
    return ((uintptr_t)p & 15) || st % per || sh % per || st < 0 || sh < 0;
}

// Few queries per segment: keys and values are read where they lie, once for each query, without images.  64 segments of 8192
// keys, 8 heads of 128, bf16 (us, images against few): 1 query each 1347 / 376, 4 each 1349 / 652, 8 each 1369 / 1088; 50 000
// keys, 8 heads over 2 key heads of 128: 4 queries 60 / 53, 8 queries 60 / 73.
inline bool attn_is_few(const MgnAttn& a) { return a.n_q <= 4 * (int64_t)a.n_seg; }

inline int attn_few_chunk(const MgnAttn& a) {                           // query heads that share a pass over a key head
    const int rep = a.heads / a.kv_heads;
    return rep >= 8 ? 8 : rep > 2 ? 4 : rep;
}
inline int64_t attn_few_blocks(const MgnAttn& a) {
    const int rep = a.heads / a.kv_heads, c = attn_few_chunk(a);
    return a.n_q * a.kv_heads * ((rep + c - 1) / c);
}

// A launch has fewer than 2^32 threads: 2^24 - 1 workgroups of 256.  What the entry point would launch for these counts, at most (a
// grid of tiles has one more per segment; images take four (head, subtile) pairs to a workgroup).
inline bool attn_launches(const MgnAttn& a, bool backward) {
    const int64_t most = (1 << 24) - 1, q_images = (a.n_q / 32 + a.n_seg) * (int64_t)a.heads, k_images = (a.n_k / 32 + a.n_seg) * (int64_t)a.kv_heads;
    const int64_t q_tiles = (a.n_q / 128 + a.n_seg) * (int64_t)a.heads, k_tiles = (a.n_k / 128 + a.n_seg) * (int64_t)a.kv_heads;
    if (backward) return q_images + k_images <= 2 * most && q_tiles <= most && k_tiles <= most;
    if (attn_is_few(a)) return attn_few_blocks(a) <= most;
    return k_images <= 2 * most && q_tiles <= most;
}

inline int attn_check(const MgnAttn* a, const char* name, bool backward) {
    const char* bad = nullptr;
    if (!a) bad = "null arguments";
    else if (a->dtype != MGN_F32 && a->dtype != MGN_BF16 && a->dtype != MGN_F16) bad = "unknown type";
    else if (a->dim < 8 || a->dim > 128 || a->dim % 8) bad = "the head width must be a multiple of 8 up to 128";
    else if (a->heads < 1 || a->kv_heads < 1 || a->heads > 1024 || a->heads % a->kv_heads) bad = "heads must be a multiple of kv_heads, 1024 at most";
    else if (a->n_q < 0 || a->n_k < 0 || a->n_q > 0x7fffffffLL - 4096 || a->n_k > 0x7fffffffLL - 4096) bad = "token counts must fit 32 bits";
    else if (a->n_seg < 1 || a->n_seg > (1 << 20) || (a->n_seg > 1 && (!a->q_ptr || !a->k_ptr))) bad = "more than one segment needs both offset arrays";
    else if ((a->q_ptr == nullptr) != (a->k_ptr == nullptr)) bad = "segment offsets come for queries and keys, or for neither";
    else if (!(a->scale > 0.f) || !std::isfinite(a->scale)) bad = "the scale must be positive and finite";
    else if ((a->n_q > 0 && !a->q) || (a->n_k > 0 && (!a->k || !a->v))) bad = "null operand";
    else if ((a->n_q > 0 && attn_bad_rows(a->q, a->q_st, a->q_sh, a->dtype)) ||
             (a->n_k > 0 && (attn_bad_rows(a->k, a->k_st, a->k_sh, a->dtype) || attn_bad_rows(a->v, a->v_st, a->v_sh, a->dtype))))
        bad = "rows must start on 16-byte borders";
    else if ((a->n_q / 32 + a->n_seg) * (int64_t)a->heads > 0x3fffffffLL || (a->n_k / 32 + a->n_seg) * (int64_t)a->kv_heads > 0x3fffffffLL)
        bad = "too many tokens x heads";
    else if (!attn_launches(*a, backward)) bad = "too many (segments + tokens / 128) x heads for one launch";
    else if (a->bias_table) {
        if (!a->bucket_lut || (a->n_q > 0 && !a->q_pos) || (a->n_k > 0 && !a->k_pos)) bad = "the bias needs a bucket table and places";
        else if (a->axes < 1 || a->axes > 3) bad = "places have one to three axes";
        else if (a->reach < 1 || a->reach > ATT_MAX_REACH) bad = "reach must be 1 .. 1024";
        else if (a->n_bucket < 1 || a->n_bucket > ATT_MAX_BUCKETS) bad = "1 .. 64 buckets";
    }
    if (bad) { mgn_set_error("%s: %s", name, bad); return MGN_E_ARG; }
    return 0;
}

// Small problems: 32 queries of a head per workgroup and no images, one launch instead of two.  It converts a subtile anew in
// every workgroup, so it pays while all workgroups are resident at once, a workgroup's chain of subtiles is short and there is
// little work in all (us, images against small): fp32, 4 heads of 32: 561 x 280 16.1 / 12.1, 4000 x 1000 26.3 / 26.1, 6000 x 300
// 16.2 / 18.7, 12 000 x 150 16.5 / 23.4, 100 000 x 20 31 / 114, 500 x 2000 21.7 / 37.3, 7900 x 2000 49 / 88; 8 heads of 64: 500 x
// 500 24.9 / 17.6, 4000 x 500 27.1 / 65.7, fp16, 500 x 250 16.6 / 15.5; bf16, 4 heads of 32: 500 x 500 16.1 / 13.7, 500 x 1000 18.9 /
// 24.1; 4 heads of 128: 500 x 250 17.5 / 20.5.
inline bool attn_is_small(const MgnAttn& a) {
    const int64_t chain = a.n_k / a.n_seg * attn_dp(a.dim), blocks = (a.n_q / 32 + a.n_seg) * (int64_t)a.heads;
    return blocks <= 512 && chain <= (a.dtype == MGN_F32 ? 32768 : 16384) && blocks * chain <= 1 << 24;
}

// Split key ranges until there are about four workgroups per compute unit, in pieces of at least 256 keys (within 3 % of two or
// eight workgroups, and of 128 keys; pieces of 512 keys take 30 instead of 26.5 us for one query over 100 000 keys in fp32).
inline int attn_few_splits(const MgnAttn& a) {
    const int64_t blocks = attn_few_blocks(a), keys = a.n_k / a.n_seg;
    int64_t s = blocks > 0 ? 1024 / blocks : 1;
    if (s > keys / 256) s = keys / 256;
    return (int)(s < 1 ? 1 : s > ATT_MAX_SPLITS ? ATT_MAX_SPLITS : s);
}
// Eight waves share the images of a tile of keys where 256 queries per workgroup still reach every compute unit.  Width 128,
// 16 bits (us, four waves against eight): 8192 x 8192 318 / 290, 4096 x 8192 181 / 169, 32 768 x 1024 173 / 179.
inline int attn_fwd_waves(const MgnAttn& a) {
    return !a.bias_table && attn_dp(a.dim) == 128 && a.dtype != MGN_F32 && (a.n_q / 256 + a.n_seg) * a.heads >= 256 ? 8 : 4;
}
// Two heads per wave of the tiled kernel share the places of a lattice, where the registers hold them and four workgroups per
// compute unit are there to begin with (100 000 x 1225, 4 heads of 32, plane: fp32 382 -> 364 us, fp16 298 -> 243; of 64, fp16
// 380 -> 321; 32 768 queries, fp32, 132 -> 115).  A place on a line is too cheap to share (295 us alone, 316 shared), and two
// heads of 64 in fp32 spill.
inline int attn_fwd_share(const MgnAttn& a) {
    return a.bias_table && a.axes > 1 && attn_dp(a.dim) <= (a.dtype == MGN_F32 ? 32 : 64) && a.heads % 2 == 0 &&
           (a.n_q / ATT_TQ + a.n_seg) * a.heads >= 1024 ? 2 : 1;
}
// Workgroups that are all resident at once and take equally long finish in whole rounds: 628 of them on 256 compute units take
// three rounds' time for two and a half rounds' work.  Key ranges are split once more where that fills the rounds better by a
// tenth and leaves 1024 keys to each piece, so that joining the pieces stays cheap (20 000 x 2501, 4 heads of 32, fp32: forward
// 206 -> 188 us with the join; 1800 x 1800, 8 heads of 64, four segments, would have gone from 77 to 78).
inline int attn_round_splits(int64_t blocks, int64_t keys, int64_t s) {
    if (blocks <= 0 || blocks * s > 1024) return (int)s;
    auto rounds = [&](int64_t n) { return (double)((blocks * n + 255) / 256) / (double)n; };
    int64_t best = s;
    for (int64_t n = s + 1; n <= 2 * s && n <= keys / 1024; ++n)
        if (rounds(n) < 0.9 * rounds(best)) best = n;
    return (int)best;
}
// workgroups of `rows` tokens in ragged segments: exact for one segment, the mean for several
inline int64_t attn_tiles(int64_t T, int64_t n_seg, int64_t rows) { return (T + rows - 1) / rows + (n_seg - 1) / 2; }
// Key ranges are split as for few queries when the query tiles leave compute units idle.
inline int attn_fwd_splits(const MgnAttn& a) {
    const int64_t blocks = attn_tiles(a.n_q, a.n_seg, 32 * attn_fwd_waves(a)) * (a.heads / attn_fwd_share(a)), keys = a.n_k / a.n_seg;
    int64_t s = blocks > 0 ? 2048 / (blocks * attn_fwd_waves(a)) : 1;
    if (s > keys / 256) s = keys / 256;
    return attn_round_splits(blocks, keys, s < 1 ? 1 : s > 64 ? 64 : s);
}

}  // namespace
