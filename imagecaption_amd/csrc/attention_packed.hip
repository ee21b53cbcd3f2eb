// Attention over packed sequences: rows of sequences of different lengths back to back in one matrix, grouped heads (Hq
// query heads share Hkv key / value heads), causal or not, with its backward.  See include/capdec.h (capdec_attn_packed_*).
//
//   s_ij = scale q_i . k_j  (causal: j <= i + nk - nq),  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i;  dp_ij = do_i . v_j;  ds_ij = p_ij (dp_ij - do_i . o_i)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i, both sums over the query heads of the group
//
// A workgroup of NW waves owns NW x 32 rows of one head (a wave owns 32: one row on a lane and its partner lane ^ 32) and
// walks the other side's rows in tiles that all its waves read from LDS; the next tile travels global -> registers while
// the current one is multiplied.  Tiles come from a table made once per set of lengths on the host, longest first, so no
// workgroup searches for its sequence and the tail of a launch is made of its shortest tiles.  What a row sums up
// stays inside one workgroup, or is joined in a fixed order: no atomics, bitwise reproducible.  The backward runs twice over the scores (dq by query
// tiles, dk / dv by key tiles and all heads of the group): 7 products instead of 5, in exchange for no fp32 gradient
// block in memory and no order that depends on the launch.
#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "attention_tile.h"

namespace capdec {

struct PackedItem {  // one tile of rows of one sequence
    int q0, nq, k0, nk;  // the sequence's rows in the packed matrices
    int t0;              // first row of this tile within its side
    int reserved[3];
};

constexpr int WALK_LEVELS = 5;

struct PackedParams {
    const void* q; const void* k; const void* v; const void* o; const void* dout;
    void* out; void* dq; void* dk; void* dv;
    float* lse; float* delta;
    void* stats;  // bf16 matrices: 16 bytes for each (head, row), see packed16_bwd_dkv_kernel
    const PackedItem* items;
    int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    int Hq, Hkv, group, causal;
    size_t stat_rows;  // rows of one head in lse / delta
    float scale;
    int parts, slots;          // dk, dv: parts of the longest key tiles (1: no tile is split), partial sums of one head
    int levels[WALK_LEVELS];   // tiles whose walk is longer than 1/2, 1/4, .. of the longest: parts, parts / 2, .. each
    float* part;               // partial sums [Hkv, slots, dk | dv, 64 keys, dh]
};

// workgroup -> (head, item): with heads in eights every XCD (blockIdx % 8) serves its own run of neighbouring heads, so
// the key / value rows of a group are fetched into one L2; items stay in the table's order (longest first)
__device__ __forceinline__ void packed_place(int heads, int& head, int& item) {
    const int blk = blockIdx.x;
    if (heads % 8 == 0) {
        const int per = heads >> 3, idx = blk >> 3;
        head = (blk & 7) * per + idx % per;
        item = idx / per;
    } else {
        head = blk % heads;
        item = blk / heads;
    }
}

// index in the list of key tiles with their parts -> tile, part of its walk, parts of it
__device__ __forceinline__ void walk_part(const PackedParams& p, int at, int& item, int& part, int& parts) {
    item = part = 0;
    parts = 1;
#pragma unroll
    for (int l = 0; l < WALK_LEVELS; ++l) {
        const int cut = p.parts >> l, n = p.levels[l];
        if (cut <= 1) break;
        if (at < n * cut) {
            item += at / cut;
            part = at % cut;
            parts = cut;
            return;
        }
        at -= n * cut;
        item += n;
    }
    item += at;
}

// accumulators of a wave through LDS to another wave with the same lane layout
template <int NDT>
__device__ __forceinline__ void put_sums(unsigned char* box, const f32x16* acc, int lane) {
#pragma unroll
    for (int i = 0; i < 4 * NDT; ++i) {
        const f32x16& a = acc[i >> 2];
        const int e = 4 * (i & 3);
        reinterpret_cast<f32x4t*>(box)[i * 64 + lane] = f32x4t{a[e], a[e + 1], a[e + 2], a[e + 3]};
    }
}
// acc = acc fa + box fb
template <int NDT>
__device__ __forceinline__ void add_sums(const unsigned char* box, f32x16* acc, int lane, float fa, float fb) {
#pragma unroll
    for (int i = 0; i < 4 * NDT; ++i) {
        const f32x4t v = reinterpret_cast<const f32x4t*>(box)[i * 64 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i >> 2][4 * (i & 3) + j] = acc[i >> 2][4 * (i & 3) + j] * fa + v[j] * fb;
    }
}

// (One wave a workgroup: bound by the way from launch to store, so the weights can keep 16 bits.  With bf16 weights alone the
// result is off by 0.0023 of itself instead of the 0.0017 that its own rounding makes; 256 captions, forward 6.1 -> 6.2 us, backward
// 9.8 -> 10.7.)
// RB blocks of 32 rows; the KS waves of a block take every KS-th run of 32 KB keys of a tile and join at the end.  ONE: no walk is
// longer than one tile, so there is one pair of images (132 sequences of 2 tokens, 15 heads of 128, fp32: 38 us with two, 19 with
// one)
template <typename T, int DH, int RB, int KS, int KB, bool ONE = false>
__global__ __launch_bounds__(RB * KS * 64, RB * KS == 4 ? 2 : 1) void packed_fwd_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int NT = RB * KS * 64, BN = 32 * KB * KS, IMG = BN * L::ROWB, BOX = (DH / 8 * 16 + 8) * 64;
    constexpr int JOIN = RB * (KS - 1) * BOX, IMAGES = ONE ? 2 : 4;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[IMAGES * IMG > JOIN ? IMAGES * IMG : JOIN];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int rb = wave % RB, ksp = wave / RB;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const T* qg = (const T*)p.q + (size_t)w.q0 * p.ldq + head * DH;
    const T* kg = (const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const T* vg = (const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + rb * 32;                // this wave's first row
    const int row = r0 + l31, off = w.nk - w.nq;  // causal: row sees keys j <= row + off
    const int kmax = p.causal ? min(w.nk, min(w.t0 + RB * 32, w.nq) + off) : w.nk;  // of the workgroup's last row
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    // keys the wave's rows can see at all, and keys that all of them see (no mask below)
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;

    typename L::frag qf[L::NF];
    L::load_row(qf, qg + (size_t)row * p.ldq, row < w.nq, half);
    Staged<T, DH, NT, BN> ks, vs;
    if (nt > 0) {
        ks.load(kg, p.ldk, 0, w.nk, tid);
        vs.load(vg, p.ldv, 0, w.nk, tid);
        ks.store(smem, tid);
        vs.store(smem + IMG, tid);
    }
    typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    Running run;
    run.init();
    landed(qf);
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const unsigned char* Ks = smem + (t & 1) * 2 * IMG + ksp * 32 * KB * L::ROWB;
        const unsigned char* Vs = Ks + IMG;
        const bool more = !ONE && t + 1 < nt;
        if (more) {
            ks.load(kg, p.ldk, (t + 1) * BN, w.nk, tid);
            vs.load(vg, p.ldv, (t + 1) * BN, w.nk, tid);
        }
        __builtin_amdgcn_sched_barrier(0);
        renew<DH>(ln);
        const int k0 = t * BN + ksp * 32 * KB;
        if (k0 < wave_end) {
            f32x16 s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                zero16(s[b]);
                L::mma_rows(s[b], Ks + b * 32 * L::ROWB, ln, qf);  // S^T[key][query]
            }
            if (k0 + 32 * KB > all_see) {
                const int see = p.causal ? min(w.nk, row + 1 + off) : w.nk;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] = k0 + 32 * b + row_of(r, half) < see ? s[b][r] : -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
            bool raised;
            const float a = run.raise(top, c, &raised);
            if (raised) {
#pragma unroll
                for (int dt = 0; dt < L::NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[dt][r] *= a;
            }
            const float base = run.base();
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[r] = exp2_fast(__fmaf_rn(s[b][r], c, -base));
                    run.l += x[r];
                }
                std::conditional_t<RB * KS == 1, typename L::weights2, typename L::weights> pw;
                L::pack(pw, x);
                if constexpr (ONE) L::mma_cols(acc, Vs, ln, pw, w.nk);
                else L::mma_cols(acc, Vs + b * 32 * L::ROWB, ln, pw);  // O^T[dim][query] += V^T P^T
            }
        }
        if (more) {
            unsigned char* nx = smem + ((t + 1) & 1) * 2 * IMG;
            ks.store(nx, tid);
            vs.store(nx + IMG, tid);
            __syncthreads();
        }
    }
    float l = run.l + __shfl_xor(run.l, 32, 64);
    if constexpr (KS > 1) {  // the later waves of a block hand their part to the first, which joins them in order
        __syncthreads();
        if (ksp > 0) {
            unsigned char* box = smem + (rb * (KS - 1) + ksp - 1) * BOX;
            put_sums<L::NDT>(box, acc, lane);
            reinterpret_cast<float2*>(box + DH / 8 * 16 * 64)[lane] = float2{run.m2, l};
        }
        __syncthreads();
        if (ksp > 0) return;
#pragma unroll
        for (int o = 0; o < KS - 1; ++o) {
            const unsigned char* box = smem + (rb * (KS - 1) + o) * BOX;
            const float2 ml = reinterpret_cast<const float2*>(box + DH / 8 * 16 * 64)[lane];
            const float m = fmaxf(run.m2, ml.x);
            const float fa = run.m2 == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(run.m2 - m);
            const float fb = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_fast(ml.x - m);
            l = l * fa + ml.y * fb;
            run.m2 = m;
            add_sums<L::NDT>(box, acc, lane, fa, fb);
        }
    }
    if (row < w.nq) {
        const bool any = l != 0.f;  // (NaN too: such a row is not an empty one)
        L::store_row((T*)p.out + (size_t)(w.q0 + row) * p.ldo + head * DH, acc, any ? 1.f / l : 0.f, half);
        if (p.lse && half == 0)
            p.lse[(size_t)head * p.stat_rows + w.q0 + row] = any ? (run.base() + __log2f(l)) * LN2 : -INFINITY;
    }
}

// The forward of bf16 matrices with 128 rows a workgroup: 64 keys at a time by DMA, one tile ahead.  Registers for the tile
// on its way would leave none for reading LDS ahead of the matrix instructions.
template <int DH>
__global__ __launch_bounds__(256, 2) void packed16_fwd_kernel(PackedParams p) {
    using L = DmaTile<DH>;
    constexpr int KB = 2, BN = 32 * KB, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const __bf16* kg = (const __bf16*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const __bf16* vg = (const __bf16*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + wave * 32;              // this wave's first row
    const int row = r0 + l31, off = w.nk - w.nq;  // causal: row sees keys j <= row + off
    const int kmax = p.causal ? min(w.nk, min(w.t0 + 128, w.nq) + off) : w.nk;  // of the workgroup's last row
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    // keys the wave's rows can see at all, and keys that all of them see (no mask below)
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;
    typename L::frag qf[L::NF];
    L::load_row(qf, (const __bf16*)p.q + (size_t)(w.q0 + row) * p.ldq + head * DH, row < w.nq, half);
    landed(qf);
    typename L::template Fetch<BN, 4> fk, fv;
    fk.init(p.ldk, lane);
    fv.init(p.ldv, lane);
    if (nt > 0) {
        fk(smem, kg, p.ldk, 0, w.nk, wave, lane);
        fv(smem + IMG, vg, p.ldv, 0, w.nk, wave, lane);
    }
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    Running run;
    run.init();
    // the two images are two copies of the loop's body: their LDS addresses are constants
    auto turn = [&](int t, unsigned char* cur, unsigned char* nx) __attribute__((always_inline)) {
        const unsigned char* Ks = cur;
        const unsigned char* Vs = Ks + IMG;
        dma_sync();
        if (t + 1 < nt) {
            fk(nx, kg, p.ldk, (t + 1) * BN, w.nk, wave, lane);
            fv(nx + IMG, vg, p.ldv, (t + 1) * BN, w.nk, wave, lane);
        }
        const int k0 = t * BN;
        if (k0 < wave_end) {
            f32x16 s[KB];
            bf16x8t kf[KB][L::NF], vf[2 * L::NDT];
#pragma unroll
            for (int b = 0; b < KB; ++b) L::read_rows(kf[b], Ks + b * 32 * L::ROWB, ln);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int b = 0; b < KB; ++b) zero16(s[b]);
#pragma unroll
            for (int ks = 0; ks < L::NF; ++ks)
#pragma unroll
                for (int b = 0; b < KB; ++b)
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[b][ks], qf[ks], s[b], 0, 0, 0);  // S^T[key][query]
            __builtin_amdgcn_s_setprio(0);
            L::read_cols(vf, Vs, ln);
            __builtin_amdgcn_sched_barrier(0);
            if (k0 + BN > all_see) {
                const int see = p.causal ? min(w.nk, row + 1 + off) : w.nk;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] = k0 + 32 * b + row_of(r, half) < see ? s[b][r] : -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
            bool raised;
            const float a = run.raise(top, c, &raised);
            if (raised) {
#pragma unroll
                for (int dt = 0; dt < L::NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[dt][r] *= a;
            }
            const float base = run.base();
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[r] = exp2_fast(__fmaf_rn(s[b][r], c, -base));
                    run.l += x[r];
                }
                typename L::weights pw;
                L::pack(pw, x);
                L::mma_read_cols(acc, vf, pw);  // O^T[dim][query] += V^T P^T
                if (b + 1 < KB) L::read_cols(vf, Vs + (b + 1) * 32 * L::ROWB, ln);
            }
        }
    };
    for (int t = 0; t < nt; t += 2) {
        turn(t, smem, smem + 2 * IMG);
        if (t + 1 < nt) turn(t + 1, smem + 2 * IMG, smem);
    }
    const float l = run.l + __shfl_xor(run.l, 32, 64);
    if (row < w.nq) {
        const bool any = l != 0.f;  // (NaN too: such a row is not an empty one)
        L::store_row((__bf16*)p.out + (size_t)(w.q0 + row) * p.ldo + head * DH, acc, any ? 1.f / l : 0.f, half);
        if (p.lse && half == 0)
            p.lse[(size_t)head * p.stat_rows + w.q0 + row] = any ? (run.base() + __log2f(l)) * LN2 : -INFINITY;
    }
}

// rowsum(do * o) of this lane's row, whose do fragments stay in df
template <typename T, int DH>
__device__ __forceinline__ float row_delta(const PackedParams& p, typename AttTile<T, DH>::frag* df, size_t grow, int head, bool mine, int half) {
    using L = AttTile<T, DH>;
    typename L::frag of[L::NF];
    L::load_row(of, (const T*)p.o + grow * p.ldo + head * DH, mine, half);
    L::load_row(df, (const T*)p.dout + grow * p.lddo + head * DH, mine, half);
    const float d = L::dot(df, of);
    return d + __shfl_xor(d, 32, 64);
}

// lse times log2 e of this lane's row: p = exp2(s c - lse2); a row that sees nothing has lse = -inf, its weights are zeros
__device__ __forceinline__ float row_lse2(const PackedParams& p, size_t grow, int head, bool mine) {
    const float lse2 = mine ? p.lse[(size_t)head * p.stat_rows + grow] * LOG2E : INFINITY;
    return lse2 == -INFINITY ? INFINITY : lse2;
}

// the row's statistics for the dk / dv kernel
template <typename T>
__device__ __forceinline__ void leave_stats(const PackedParams& p, float lse2, float dsum, size_t grow, int head) {
    const size_t at = (size_t)head * p.stat_rows + grow;
    if (sizeof(T) == 2 && p.stats) {
        // -lse / scale and -delta, three bf16 terms each; a row that sees nothing gets weights of zero
        const float l = lse2 == INFINITY ? -1e30f : -lse2 / (p.scale * LOG2E), d = -dsum;
        const __bf16 l0 = (__bf16)l, l1 = (__bf16)(l - (float)l0), l2 = (__bf16)(l - (float)l0 - (float)l1);
        const __bf16 d0 = (__bf16)d, d1 = (__bf16)(d - (float)d0), d2 = (__bf16)(d - (float)d0 - (float)d1);
        reinterpret_cast<bf16x8t*>(p.stats)[at] = bf16x8t{l0, l1, l2, (__bf16)0.f, d0, d1, d2, (__bf16)0.f};
    } else {
        p.delta[at] = dsum;
    }
}

// Score gradients of one block: x = p (dp - delta).  Rows whose keys all lie in this block take delta = sum p dp from the
// block itself: from the rounded o it is off by 2^-9 |do . o|, which is all that dq and dk of such rows consist of when they
// see one key (their true value is zero) and more than the other roundings when they see a few.
__device__ __forceinline__ void score_grads(float* x, const f32x16& s, const f32x16& dp, float c, float lse2, bool one_block, float& dsum) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = exp2_fast(__fmaf_rn(s[r], c, -lse2));
    if (one_block) {
        float d = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) d = __fmaf_rn(x[r], x[r] > 0.f ? dp[r] : 0.f, d);
        dsum = d + __shfl_xor(d, 32, 64);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= dp[r] - dsum;
}

// dq and delta = rowsum(do * o); blocks and waves as in the forward
template <typename T, int DH, int RB, int KS, int KB>
__global__ __launch_bounds__(RB * KS * 64, RB * KS == 4 && (sizeof(T) == 2 || DH == 64) ? 2 : 1) void packed_bwd_dq_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int NT = RB * KS * 64, BN = 32 * KB * KS, IMG = BN * L::ROWB, BOX = DH / 8 * 16 * 64;
    constexpr int JOIN = RB * (KS - 1) * BOX;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG > JOIN ? 4 * IMG : JOIN];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int rb = wave % RB, ksp = wave / RB;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const T* kg = (const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const T* vg = (const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + rb * 32;
    const int row = r0 + l31, off = w.nk - w.nq;
    const int kmax = p.causal ? min(w.nk, min(w.t0 + RB * 32, w.nq) + off) : w.nk;
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;
    const bool mine = row < w.nq;
    const size_t grow = (size_t)(w.q0 + row);

    Staged<T, DH, NT, BN> ks, vs;
    if (nt > 0) {
        ks.load(kg, p.ldk, 0, w.nk, tid);
        vs.load(vg, p.ldv, 0, w.nk, tid);
    }
    typename L::frag qf[L::NF], df[L::NF];
    float dsum = row_delta<T, DH>(p, df, grow, head, mine, half);
    L::load_row(qf, (const T*)p.q + grow * p.ldq + head * DH, mine, half);
    const float lse2 = row_lse2(p, grow, head, mine);
    const bool one_block = wave_end <= 32;
    if (nt > 0) {
        ks.store(smem, tid);
        vs.store(smem + IMG, tid);
    }
    typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    landed(qf);
    landed(df);
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const unsigned char* Ks = smem + (t & 1) * 2 * IMG + ksp * 32 * KB * L::ROWB;
        const unsigned char* Vs = Ks + IMG;
        const bool more = t + 1 < nt;
        if (more) {
            ks.load(kg, p.ldk, (t + 1) * BN, w.nk, tid);
            vs.load(vg, p.ldv, (t + 1) * BN, w.nk, tid);
        }
        __builtin_amdgcn_sched_barrier(0);
        renew<DH>(ln);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int k0 = t * BN + (ksp * KB + b) * 32;
            if (k0 < wave_end) {
                f32x16 s, dp;
                zero16(s);
                zero16(dp);
                L::mma_rows(s, Ks + b * 32 * L::ROWB, ln, qf);   // S^T[key][query]
                L::mma_rows(dp, Vs + b * 32 * L::ROWB, ln, df);  // dP^T[key][query]
                if (k0 + 32 > all_see) {
                    const int see = p.causal ? min(w.nk, row + 1 + off) : w.nk;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = k0 + row_of(r, half) < see ? s[r] : -INFINITY;
                }
                float x[16];
                score_grads(x, s, dp, c, lse2, one_block, dsum);
                typename L::weights dw;
                L::pack(dw, x);
                L::mma_cols(acc, Ks + b * 32 * L::ROWB, ln, dw);  // dQ^T[dim][query] += K^T dS^T
            }
        }
        if (more) {
            unsigned char* nx = smem + ((t + 1) & 1) * 2 * IMG;
            ks.store(nx, tid);
            vs.store(nx + IMG, tid);
            __syncthreads();
        }
    }
    if constexpr (KS > 1) {
        __syncthreads();
        if (ksp > 0) put_sums<L::NDT>(smem + (rb * (KS - 1) + ksp - 1) * BOX, acc, lane);
        __syncthreads();
        if (ksp > 0) return;
#pragma unroll
        for (int o = 0; o < KS - 1; ++o) add_sums<L::NDT>(smem + (rb * (KS - 1) + o) * BOX, acc, lane, 1.f, 1.f);
    }
    if (mine) {
        L::store_row((T*)p.dq + grow * p.lddq + head * DH, acc, p.scale, half);
        if (half == 0) leave_stats<T>(p, lse2, dsum, grow, head);
    }
}

// dq of bf16 matrices with 128 rows a workgroup, fed as the forward is
template <int DH>
__global__ __launch_bounds__(256, 2) void packed16_bwd_dq_kernel(PackedParams p) {
    using L = DmaTile<DH>;
    constexpr int KB = 2, BN = 32 * KB, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const __bf16* kg = (const __bf16*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const __bf16* vg = (const __bf16*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + wave * 32;
    const int row = r0 + l31, off = w.nk - w.nq;
    const int kmax = p.causal ? min(w.nk, min(w.t0 + 128, w.nq) + off) : w.nk;
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;
    const bool mine = row < w.nq;
    const size_t grow = (size_t)(w.q0 + row);
    typename L::template Fetch<BN, 4> fk, fv;
    fk.init(p.ldk, lane);
    fv.init(p.ldv, lane);
    if (nt > 0) {
        fk(smem, kg, p.ldk, 0, w.nk, wave, lane);
        fv(smem + IMG, vg, p.ldv, 0, w.nk, wave, lane);
    }
    typename L::frag qf[L::NF], df[L::NF];
    float dsum = row_delta<__bf16, DH>(p, df, grow, head, mine, half);
    L::load_row(qf, (const __bf16*)p.q + grow * p.ldq + head * DH, mine, half);
    const float lse2 = row_lse2(p, grow, head, mine);
    const bool one_block = wave_end <= 32;
    landed(qf);
    typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    auto turn = [&](int t, unsigned char* cur, unsigned char* nx) __attribute__((always_inline)) {
        const unsigned char* Ks = cur;
        const unsigned char* Vs = Ks + IMG;
        dma_sync();
        if (t + 1 < nt) {
            fk(nx, kg, p.ldk, (t + 1) * BN, w.nk, wave, lane);
            fv(nx + IMG, vg, p.ldv, (t + 1) * BN, w.nk, wave, lane);
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int k0 = t * BN + 32 * b;
            if (k0 < wave_end) {
                f32x16 s, dp;
                zero16(s);
                zero16(dp);
                __builtin_amdgcn_s_setprio(1);
                L::mma_rows(s, Ks + b * 32 * L::ROWB, ln, qf);   // S^T[key][query]
                L::mma_rows(dp, Vs + b * 32 * L::ROWB, ln, df);  // dP^T[key][query]
                __builtin_amdgcn_s_setprio(0);
                if (k0 + 32 > all_see) {
                    const int see = p.causal ? min(w.nk, row + 1 + off) : w.nk;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = k0 + row_of(r, half) < see ? s[r] : -INFINITY;
                }
                float x[16];
                score_grads(x, s, dp, c, lse2, one_block, dsum);
                typename L::weights dw;
                L::pack(dw, x);
                L::mma_cols(acc, Ks + b * 32 * L::ROWB, ln, dw);  // dQ^T[dim][query] += K^T dS^T
            }
        }
    };
    for (int t = 0; t < nt; t += 2) {
        turn(t, smem, smem + 2 * IMG);
        if (t + 1 < nt) turn(t + 1, smem + 2 * IMG, smem);
    }
    if (mine) {
        L::store_row((__bf16*)p.dq + grow * p.lddq + head * DH, acc, p.scale, half);
        if (half == 0) leave_stats<__bf16>(p, lse2, dsum, grow, head);
    }
}

// dq, dk, dv of sequences that fit one block of 32 rows on both sides, in one pass: a workgroup takes a (sequence, key / value
// head), its W waves every W-th query head of the group, and the first wave adds up their dk and dv in order.  Everything is
// read once and o not at all (delta = sum p dp, see score_grads).  Scores are made once, keys x queries; dk and dv, which sum
// over the queries, take the transposed weights through LDS.  Products over the rows of an image stop behind the last one.
// Weights keep 16 bits, as in the forward.  256 captions of up to 20 tokens, 8 heads of 64: bf16 10.0 us (dq, then dk and dv: 14.5;
// scores made in both orientations instead of weights transposed: 10.3), fp32 26 (29); 64 sequences of 10 to 30 tokens, 32 heads
// of 128 over 4, bf16: 19, 40 with one wave for the group.
template <typename T, int DH, int W>
__global__ __launch_bounds__(64 * W, DH == 64 && sizeof(T) == 2 ? 2 : 1) void packed_bwd_block_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int IMG = 32 * L::ROWB, BOX = DH / 8 * 16 * 64, TURN = 33;
    constexpr bool AHEAD = L::ROWB <= 256;  // a wider head's rows on their way would not fit the registers
    static_assert(BOX <= 2 * IMG, "a wave's sums fit its images");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[(2 + 2 * W) * IMG];
    __shared__ float turned[W > 1 ? W : 1][W > 1 ? 32 * TURN : 1];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int hk, it;
    packed_place(p.Hkv, hk, it);
    const PackedItem w = p.items[it];
    const int off = w.nk - w.nq;  // causal: query i sees the keys j <= i + off
    const bool mine_q = l31 < w.nq, mine_k = l31 < w.nk;
    unsigned char *Ks = smem, *Vs = smem + IMG, *Qs = smem + (2 + 2 * wave) * IMG, *Ds = Qs + IMG;
    float* turn = W > 1 ? turned[wave] : reinterpret_cast<float*>(Ks);  // (one head: K and V are no longer needed then)
    Staged<T, DH, 64 * W, 32> ks, vs;
    Staged<T, DH, 64, 32> qst, dst;
    float next;
    auto fetch = [&](int g) {
        const int head = hk * p.group + g;
        qst.load((const T*)p.q + (size_t)w.q0 * p.ldq + head * DH, p.ldq, 0, w.nq, lane);
        dst.load((const T*)p.dout + (size_t)w.q0 * p.lddo + head * DH, p.lddo, 0, w.nq, lane);
        next = row_lse2(p, (size_t)(w.q0 + l31), head, mine_q);
    };
    ks.load((const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH, p.ldk, 0, w.nk, tid);
    vs.load((const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH, p.ldv, 0, w.nk, tid);
    if (AHEAD && wave < p.group) fetch(wave);
    ks.store(Ks, tid);
    vs.store(Vs, tid);
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    const int see = p.causal ? min(w.nk, l31 + 1 + off) : w.nk;
    f32x16 dk[L::NDT], dv[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) {
        zero16(dk[dt]);
        zero16(dv[dt]);
    }
    // weights [key][query] of a lane's query -> [query][key] of a lane's key
    auto transpose = [&](float* x) {
#pragma unroll
        for (int r = 0; r < 16; ++r) turn[row_of(r, half) * TURN + l31] = x[r];
        wave_fence();
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = turn[l31 * TURN + row_of(r, half)];
        wave_fence();
    };
    __syncthreads();
    for (int g = wave; g < p.group; g += W) {
        if (!AHEAD) fetch(g);
        wave_fence();
        qst.store(Qs, lane);
        dst.store(Ds, lane);
        wave_fence();
        const float lse2 = next;
        if (AHEAD && g + W < p.group) fetch(g + W);
        f32x16 s, dp;
        zero16(s);
        zero16(dp);
        L::mma_images(s, Ks, Qs, ln);   // S^T[key][query]
        L::mma_images(dp, Vs, Ds, ln);  // dP^T[key][query]
        float x[16], y[16], dsum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = row_of(r, half) < see ? exp2_fast(__fmaf_rn(s[r], c, -lse2)) : 0.f;
            dsum = __fmaf_rn(x[r], x[r] > 0.f ? dp[r] : 0.f, dsum);
        }
        dsum += __shfl_xor(dsum, 32, 64);
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = x[r] * (dp[r] - dsum);
        typename L::weights2 pw, dw;
        L::pack(dw, y);
        f32x16 dq[L::NDT];
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt) zero16(dq[dt]);
        L::mma_cols(dq, Ks, ln, dw, w.nk);  // dQ^T[dim][query] = K^T dS^T
        if (mine_q) L::store_row((T*)p.dq + (size_t)(w.q0 + l31) * p.lddq + (hk * p.group + g) * DH, dq, p.scale, half);
        wave_fence();
        transpose(x);
        L::pack(pw, x);
        L::mma_cols(dv, Ds, ln, pw, w.nq);  // dV^T[dim][key] += dO^T P
        transpose(y);
        L::pack(dw, y);
        L::mma_cols(dk, Qs, ln, dw, w.nq);  // dK^T[dim][key] += Q^T dS
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            f32x16* acc = side ? dk : dv;
            __syncthreads();
            if (wave > 0) put_sums<L::NDT>(Qs, acc, lane);
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int o = 1; o < W; ++o) add_sums<L::NDT>(smem + (2 + 2 * o) * IMG, acc, lane, 1.f, 1.f);
            }
        }
        if (wave > 0) return;
    }
    if (mine_k) {
        L::store_row((T*)p.dk + (size_t)(w.k0 + l31) * p.lddk + hk * DH, dk, p.scale, half);
        L::store_row((T*)p.dv + (size_t)(w.k0 + l31) * p.lddv + hk * DH, dv, 1.f, half);
    }
}

// dk, dv: KB blocks of 32 key rows of one key / value head, every block walked by QS waves that take every QS-th query tile
// of every query head of the group and add up at the end.  Runs after packed_bwd_dq_kernel (reads delta).
template <typename T, int DH, int KB, int QS>
__global__ __launch_bounds__(KB * QS * 64, KB * QS == 4 && (sizeof(T) == 2 || DH == 64) ? 2 : 1) void packed_bwd_dkv_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int NT = KB * QS * 64, BN = 32 * QS, IMG = BN * L::ROWB, KIMG = 32 * KB * L::ROWB;
    constexpr bool OWN_LDS = sizeof(T) == 4 && DH == 64 && NT > 64;  // the block's own rows stay in LDS: two waves a SIMD
    constexpr int BOX = DH / 8 * 16 * 64, JOIN = KB * (QS - 1) * BOX, WALK = 2 * IMG + (OWN_LDS ? 2 * KIMG : 0);
    __shared__ __attribute__((aligned(1024))) unsigned char smem[WALK > JOIN ? WALK : JOIN];
    __shared__ float stat[2][BN];  // [lse2 | delta][query]
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int kb = wave % KB, qs = wave / KB;
    int hk, at, it, part, parts;
    packed_place(p.Hkv, hk, at);
    walk_part(p, at, it, part, parts);
    const PackedItem w = p.items[it];
    const int r0 = w.t0 + kb * 32;
    const int key = r0 + l31, off = w.nk - w.nq;
    const bool mine = key < w.nk;
    // causal: query i sees key j iff i >= j - off; the first tile that meets one of the workgroup's keys
    const int first = p.causal ? max(0, w.t0 - off) / BN : 0;
    const int per = max(0, (w.nq + BN - 1) / BN - first), all = per * p.group;
    const int begin = (int)((int64_t)all * part / parts), nt = (int)((int64_t)all * (part + 1) / parts) - begin;

    typename L::frag kf[OWN_LDS ? 1 : L::NF], vf[OWN_LDS ? 1 : L::NF];
    unsigned char* Ks = smem + 2 * IMG;
    unsigned char* Vs = Ks + KIMG;
    Staged<T, DH, NT, OWN_LDS ? 32 * KB : 64> own_k, own_v;
    if constexpr (OWN_LDS) {
        own_k.load((const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH, p.ldk, w.t0, w.nk, tid);
        own_v.load((const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH, p.ldv, w.t0, w.nk, tid);
    } else {
        L::load_row(kf, (const T*)p.k + (size_t)(w.k0 + key) * p.ldk + hk * DH, mine, half);
        L::load_row(vf, (const T*)p.v + (size_t)(w.k0 + key) * p.ldv + hk * DH, mine, half);
        landed(kf);
        landed(vf);
    }
    Staged<T, DH, NT, BN> qst, dst;
    float st = 0.f;  // threads 0 .. BN - 1: a row's lse2, the next BN: its delta
    auto fetch = [&](int i) {
        const int t = begin + i, head = hk * p.group + t / per, q0 = (first + t % per) * BN;
        qst.load((const T*)p.q + (size_t)w.q0 * p.ldq + head * DH, p.ldq, q0, w.nq, tid);
        dst.load((const T*)p.dout + (size_t)w.q0 * p.lddo + head * DH, p.lddo, q0, w.nq, tid);
        if (tid < 2 * BN) {
            const int i = q0 + tid % BN;
            const float none = tid < BN ? INFINITY : 0.f;
            const float* src = tid < BN ? p.lse : p.delta;
            st = i < w.nq ? src[(size_t)head * p.stat_rows + w.q0 + i] : none;
            if (tid < BN) {
                st *= LOG2E;
                if (st == -INFINITY) st = INFINITY;
            }
        }
    };
    if (nt > 0) fetch(0);
    if constexpr (OWN_LDS) {
        own_k.store(Ks, tid);
        own_v.store(Vs, tid);
    }
    typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 dk[L::NDT], dv[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) {
        zero16(dk[dt]);
        zero16(dv[dt]);
    }
    for (int t = 0; t < nt; ++t) {
        qst.store(smem, tid);
        dst.store(smem + IMG, tid);
        if (tid < 2 * BN) stat[tid / BN][tid % BN] = st;
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1);
        __builtin_amdgcn_sched_barrier(0);
        renew<DH>(ln);
        const int q0 = (first + (begin + t) % per) * BN + 32 * qs;
        const unsigned char* Qs = smem + 32 * qs * L::ROWB;
        const unsigned char* Ds = Qs + IMG;
        if (r0 < w.nk && q0 < w.nq && (!p.causal || r0 <= q0 + 31 + off)) {
            f32x16 s, dp;
            zero16(s);
            if constexpr (OWN_LDS) L::mma_images(s, Qs, Ks + kb * 32 * L::ROWB, ln);  // S[query][key]
            else L::mma_rows(s, Qs, ln, kf);
            // queries past the end have lse2 = +inf (weight zero); keys past the end are nobody's
            if (p.causal && q0 + off < r0 + 31) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = key <= q0 + row_of(r, half) + off ? s[r] : -INFINITY;
            }
            zero16(dp);  // dP[query][key]
            if constexpr (OWN_LDS) L::mma_images(dp, Ds, Vs + kb * 32 * L::ROWB, ln);
            else L::mma_rows(dp, Ds, ln, vf);
            float x[16], y[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4t ls = *reinterpret_cast<const f32x4t*>(&stat[0][32 * qs + 8 * i + 4 * half]);
                const f32x4t de = *reinterpret_cast<const f32x4t*>(&stat[1][32 * qs + 8 * i + 4 * half]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[4 * i + j] = exp2_fast(__fmaf_rn(s[4 * i + j], c, -ls[j]));
                    y[4 * i + j] = x[4 * i + j] * (dp[4 * i + j] - de[j]);
                }
            }
            typename L::weights pw, dw;
            L::pack(pw, x);
            L::pack(dw, y);
            L::mma_cols(dv, Ds, ln, pw);  // dV^T[dim][key] += dO^T P
            L::mma_cols(dk, Qs, ln, dw);  // dK^T[dim][key] += Q^T dS
        }
        __syncthreads();
    }
    if constexpr (QS > 1) {  // the later waves of a block hand their sums to the first, in order
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            f32x16* acc = side ? dk : dv;
            if (qs > 0) put_sums<L::NDT>(smem + (kb * (QS - 1) + qs - 1) * BOX, acc, lane);
            __syncthreads();
            if (qs == 0) {
#pragma unroll
                for (int o = 0; o < QS - 1; ++o) add_sums<L::NDT>(smem + (kb * (QS - 1) + o) * BOX, acc, lane, 1.f, 1.f);
            }
            __syncthreads();
        }
    }
    if (qs == 0 && mine && parts > 1) {
        float* to = p.part + ((((size_t)hk * p.slots + at) * 2) * 32 * KB + kb * 32 + l31) * DH;
        AttTile<float, DH>::store_row(to, dk, 1.f, half);
        AttTile<float, DH>::store_row(to + 32 * KB * DH, dv, 1.f, half);
    } else if (qs == 0 && mine) {
        L::store_row((T*)p.dk + (size_t)(w.k0 + key) * p.lddk + hk * DH, dk, p.scale, half);
        L::store_row((T*)p.dv + (size_t)(w.k0 + key) * p.lddv + hk * DH, dv, 1.f, half);
    }
}

// The same for bf16, two blocks of two waves.  Q and dO tiles travel global -> LDS by DMA,
// one tile ahead: the rows come from beyond the L2 (every query head of the group is walked), and registers for them would
// cost the second wave of a SIMD.  V fragments are read from LDS for the same reason.  Per-query statistics enter the
// products as one more k-step: -lse / scale and -delta split into three bf16 terms each (24 bits, exact to fp32) times ones,
// so a lane loads 8 bytes for its own query and no value has to be handed around in accumulator-row order.
template <int DH>
__global__ __launch_bounds__(256, 2) void packed16_bwd_dkv_kernel(PackedParams p) {
    using L = DmaTile<DH>;
    constexpr int KB = 2, QS = 2, BN = 32 * QS, IMG = BN * L::ROWB, KIMG = 32 * KB * L::ROWB;
    constexpr int BOX = DH / 8 * 16 * 64, WALK = 4 * IMG + KIMG;
    static_assert(KB * QS == 4 && KB * (QS - 1) * BOX <= WALK, "the sums of a block fit the images");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[WALK];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int kb = wave % KB, qs = wave / KB;
    int hk, at, it, part, parts;
    packed_place(p.Hkv, hk, at);
    walk_part(p, at, it, part, parts);
    const PackedItem w = p.items[it];
    const int r0 = w.t0 + kb * 32;
    const int key = r0 + l31, off = w.nk - w.nq;
    const bool mine = key < w.nk;
    // causal: query i sees key j iff i >= j - off; the first tile that meets one of the workgroup's keys
    const int first = p.causal ? max(0, w.t0 - off) / BN : 0;
    const int per = max(0, (w.nq + BN - 1) / BN - first), all = per * p.group;
    const int begin = (int)((int64_t)all * part / parts), nt = (int)((int64_t)all * (part + 1) / parts) - begin;
    unsigned char* Vs = smem + 4 * IMG;
    const s16x4t* stats = reinterpret_cast<const s16x4t*>(p.stats);
    s16x4t st;
    // the next tile to fetch: head, tile
    int fh = hk * p.group + (per ? begin / per : 0), fq = first + (per ? begin % per : 0);
    typename L::template Fetch<BN, 4> fetch_q, fetch_do;
    fetch_q.init(p.ldq, lane);
    fetch_do.init(p.lddo, lane);
    auto fetch = [&](unsigned char* to) __attribute__((always_inline)) {
        const int q0 = fq * BN;
        st = stats[2 * ((size_t)fh * p.stat_rows + w.q0 + min(q0 + 32 * qs + l31, w.nq - 1)) + half];
        fetch_q(to, (const __bf16*)p.q + (size_t)w.q0 * p.ldq + fh * DH, p.ldq, q0, w.nq, wave, lane);
        fetch_do(to + IMG, (const __bf16*)p.dout + (size_t)w.q0 * p.lddo + fh * DH, p.lddo, q0, w.nq, wave, lane);
        if (++fq == first + per) {
            fq = first;
            ++fh;
        }
    };
    typename L::frag kf[L::NF];
    L::load_row(kf, (const __bf16*)p.k + (size_t)(w.k0 + key) * p.ldk + hk * DH, mine, half);
    if (nt > 0) {
        typename L::template Fetch<32 * KB, 4> fv;
        fv.init(p.ldv, lane);
        fv(Vs, (const __bf16*)p.v + (size_t)w.k0 * p.ldv + hk * DH, p.ldv, w.t0, w.nk, wave, lane);
        fetch(smem);
    }
    typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    // half-wave 0 holds the terms of -lse / scale (k = 0..3), half-wave 1 those of -delta (k = 4..7)
    constexpr short ONE = 0x3f80;
    const short f0 = half ? 0 : ONE, f1 = half ? ONE : 0;
    const s16x4t pick_l = {f0, f0, f0, f0}, pick_d = {f1, f1, f1, f1};
    f32x16 dk[L::NDT], dv[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) {
        zero16(dk[dt]);
        zero16(dv[dt]);
    }
    landed(kf);
    int qt = first + (per ? begin % per : 0);
    for (int t = 0; t < nt; ++t) {
        dma_sync();
        s16x4t now = st;
        asm volatile("" : "+v"(now));  // taken here, where it has landed: a wait further down would include the next tile's transfers
        if (t + 1 < nt) fetch(smem + ((t + 1) & 1) * 2 * IMG);
        const int q0 = qt * BN + 32 * qs;
        if (++qt == first + per) qt = first;
        opaque(ln.row);  // addresses are made anew every turn: kept, they would take registers that the sums need
        opaque(ln.col[0]);
        opaque(ln.col[1]);
        const unsigned char* Qs = smem + (t & 1) * 2 * IMG + 32 * qs * L::ROWB;
        const unsigned char* Ds = Qs + IMG;
        if (r0 < w.nk && q0 < w.nq && (!p.causal || r0 <= q0 + 31 + off)) {
            f32x16 s, dp;
            zero16(s);
            s = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(now, pick_l, s, 0, 0, 0);
            L::mma_rows(s, Qs, ln, kf);  // S[query][key] - lse / scale
            // rows past the last query are copies of it; keys past the end are nobody's
            if ((p.causal && q0 + off < r0 + 31) || q0 + 32 > w.nq) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = q0 + row_of(r, half);
                    s[r] = i < w.nq && (!p.causal || key <= i + off) ? s[r] : -INFINITY;
                }
            }
            zero16(dp);
            dp = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(now, pick_d, dp, 0, 0, 0);
            L::mma_images(dp, Ds, Vs + kb * 32 * L::ROWB, ln);  // dP[query][key] - delta
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = exp2_fast(s[r] * c);
            typename L::weights pw, dw;
            L::pack(pw, x);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] *= dp[r];
            L::pack(dw, x);
            L::mma_cols(dv, Ds, ln, pw);  // dV^T[dim][key] += dO^T P
            L::mma_cols(dk, Qs, ln, dw);  // dK^T[dim][key] += Q^T dS
        }
    }
    // the later waves of a block hand their sums to the first, in order
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        f32x16* acc = side ? dk : dv;
        __syncthreads();
        if (qs > 0) put_sums<L::NDT>(smem + (kb * (QS - 1) + qs - 1) * BOX, acc, lane);
        __syncthreads();
        if (qs == 0) {
#pragma unroll
            for (int o = 0; o < QS - 1; ++o) add_sums<L::NDT>(smem + (kb * (QS - 1) + o) * BOX, acc, lane, 1.f, 1.f);
        }
    }
    if (qs == 0 && mine && parts > 1) {
        float* to = p.part + ((((size_t)hk * p.slots + at) * 2) * 32 * KB + kb * 32 + l31) * DH;
        AttTile<float, DH>::store_row(to, dk, 1.f, half);
        AttTile<float, DH>::store_row(to + 32 * KB * DH, dv, 1.f, half);
    } else if (qs == 0 && mine) {
        L::store_row((__bf16*)p.dk + (size_t)(w.k0 + key) * p.lddk + hk * DH, dk, p.scale, half);
        L::store_row((__bf16*)p.dv + (size_t)(w.k0 + key) * p.lddv + hk * DH, dv, 1.f, half);
    }
}

// the parts' sums of one key tile of 64 rows, in order
template <typename T, int DH>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedParams p) {
    typedef T out4 __attribute__((ext_vector_type(4)));
    constexpr int TILE = 64 * DH;
    const int hk = blockIdx.x % p.Hkv, tid = threadIdx.x;
    int it = blockIdx.x / p.Hkv, slot = 0, parts = 1, before = 0;
#pragma unroll
    for (int l = 0; l < WALK_LEVELS; ++l) {
        const int cut = p.parts >> l, n = p.levels[l];
        if (cut <= 1) break;
        if (it < before + n) {
            parts = cut;
            slot += (it - before) * cut;
            break;
        }
        before += n;
        slot += n * cut;
    }
    const PackedItem w = p.items[it];
    const float* from = p.part + ((size_t)hk * p.slots + slot) * 2 * TILE;
#pragma unroll
    for (int side = 0; side < 2; ++side)
        for (int i = tid; i < TILE / 4; i += 256) {
            const int row = i / (DH / 4), col = i % (DH / 4) * 4;
            if (w.t0 + row >= w.nk) break;
            f32x4t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int s = 0; s < parts; ++s) sum += *reinterpret_cast<const f32x4t*>(from + (size_t)(2 * s + side) * TILE + 4 * i);
            const float mul = side ? 1.f : p.scale;
            const out4 v = {(T)(sum[0] * mul), (T)(sum[1] * mul), (T)(sum[2] * mul), (T)(sum[3] * mul)};
            T* to = side ? (T*)p.dv + (size_t)(w.k0 + w.t0 + row) * p.lddv : (T*)p.dk + (size_t)(w.k0 + w.t0 + row) * p.lddk;
            *reinterpret_cast<out4*>(to + hk * DH + col) = v;
        }
}

// rows of a workgroup's tile, as the plan's table lists them for queries and then for keys
constexpr int TILE_ROWS[3] = {128, 64, 32};

static int64_t tiles_of(const int* lens, int n, int rows) {
    int64_t t = 0;
    for (int i = 0; i < n; ++i) t += (lens[i] + rows - 1) / rows;
    return t;
}

static bool lengths_ok(const int* lens, int n) {
    int64_t sum = 0;
    for (int i = 0; i < n; ++i) {
        if (lens[i] < 0) return false;
        sum += lens[i];
    }
    return sum < (1ll << 31) - 1024;  // (a tile's first row plus its height stays an int)
}

}  // namespace capdec

using namespace capdec;

extern "C" size_t capdec_packed_table_bytes(const int* lens_q, const int* lens_k, int n) {
    if (!lens_q || n <= 0 || !lengths_ok(lens_q, n) || (lens_k && !lengths_ok(lens_k, n))) return 0;
    const int* lk = lens_k ? lens_k : lens_q;
    int64_t items = 0;
    for (int rows : TILE_ROWS) items += tiles_of(lens_q, n, rows) + tiles_of(lk, n, rows);
    return (size_t)(items > 0 ? items : 1) * sizeof(PackedItem);
}

extern "C" int capdec_packed_plan(const int* lens_q, const int* lens_k, int n, int causal, void* table_dev, size_t table_bytes,
                                  capdec_packed_seqs* seqs) {
    CAPDEC_REQUIRE(lens_q && table_dev && seqs && n > 0, "capdec_packed_plan: bad arguments (n=%d)", n);
    const size_t need = capdec_packed_table_bytes(lens_q, lens_k, n);
    CAPDEC_REQUIRE(need > 0, "capdec_packed_plan: a length is negative, or the rows pass 2^31 - 1024");
    CAPDEC_REQUIRE(aligned16(table_dev), "capdec_packed_plan: the table must be 16-byte aligned");
    if (table_bytes < need) {
        set_error("capdec_packed_plan: table of %zu bytes, %zu needed", table_bytes, need);
        return CAPDEC_ERR_WORKSPACE;
    }
    const int* lk = lens_k ? lens_k : lens_q;
    try {
        std::vector<PackedItem> all;
        all.reserve(need / sizeof(PackedItem));
        int count[6] = {0, 0, 0, 0, 0, 0};
        for (int part = 0; part < 6; ++part) {  // query tiles, then key tiles
            const bool keys = part >= 3;
            const int rows = TILE_ROWS[part % 3];
            const size_t begin = all.size();
            int q0 = 0, k0 = 0;
            for (int i = 0; i < n; ++i) {
                const int nq = lens_q[i], nk = lk[i];
                for (int t0 = 0; t0 < (keys ? nk : nq); t0 += rows) all.push_back(PackedItem{q0, nq, k0, nk, t0, {0, 0, 0}});
                q0 += nq;
                k0 += nk;
            }
            auto cost = [&](const PackedItem& a) {  // tiles of 64 queries / rows of keys that the tile walks
                if (keys) return std::max(0, (a.nq + 63) / 64 - (causal ? std::max(0, a.t0 - (a.nk - a.nq)) / 64 : 0));
                return causal ? std::min(a.nk, a.t0 + rows + a.nk - a.nq) : a.nk;
            };
            std::stable_sort(all.begin() + begin, all.end(), [&](const PackedItem& a, const PackedItem& b) { return cost(a) > cost(b); });
            count[part] = (int)(all.size() - begin);
            if (part == 4) {
                const int64_t longest = count[part] ? cost(all[begin]) : 0;
                seqs->walk_max = (int)longest;
                seqs->walk_sum = 0;
                for (int l = 0; l < WALK_LEVELS; ++l) seqs->walk_levels[l] = 0;
                for (size_t i = begin; i < all.size(); ++i) {
                    const int64_t c = cost(all[i]);
                    seqs->walk_sum += c;
                    for (int l = 0; l < WALK_LEVELS; ++l)
                        if (c << (l + 1) > longest) {
                            ++seqs->walk_levels[l];
                            break;
                        }
                }
            }
        }
        if (!all.empty() && hipMemcpy(table_dev, all.data(), all.size() * sizeof(PackedItem), hipMemcpyHostToDevice) != hipSuccess) {
            set_error("capdec_packed_plan: copying the table to the device failed");
            return CAPDEC_ERR_LAUNCH;
        }
        seqs->n = n;
        seqs->causal = causal != 0;
        seqs->rows_q = seqs->rows_k = 0;
        for (int i = 0; i < n; ++i) {
            seqs->rows_q += lens_q[i];
            seqs->rows_k += lk[i];
        }
        for (int part = 0; part < 6; ++part) seqs->tiles[part] = count[part];
        seqs->one_block = 1;
        for (int i = 0; i < n; ++i)
            if (std::max(lens_q[i], lk[i]) > 32 || (lens_q[i] == 0) != (lk[i] == 0)) seqs->one_block = 0;
        seqs->table = table_dev;
    } catch (const std::exception& e) {
        set_error("capdec_packed_plan: %s", e.what());
        return CAPDEC_ERR_ARG;
    }
    return 0;
}

namespace capdec {

static bool packed_mat(const void* p, int ld, int width, int es, int rows) {
    // (a tile's rows are addressed by 32-bit offsets: 128 rows of at most 2^25 bytes)
    return rows == 0 || (p && aligned16(p) && ld >= width && ld % (16 / es) == 0 && (int64_t)ld * es <= (1 << 25));
}

static int packed_check(const char* what, const capdec_packed_seqs* s, int Hq, int Hkv, int dh, int dtype, float scale) {
    CAPDEC_REQUIRE(s && s->table, "%s: no plan", what);
    CAPDEC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "%s: Hq=%d must be a positive multiple of Hkv=%d", what, Hq, Hkv);
    CAPDEC_REQUIRE(dh == 64 || dh == 128, "%s: head dim %d not in {64,128}", what, dh);
    CAPDEC_REQUIRE(dtype == CAPDEC_F32 || dtype == CAPDEC_BF16S, "%s: dtype %d: fp32 (CAPDEC_F32) or bf16 (CAPDEC_BF16S) matrices", what, dtype);
    CAPDEC_REQUIRE(scale_ok(scale), "%s: scale must lie between 2^-60 and 2^60", what);
    CAPDEC_REQUIRE((int64_t)Hq * dh < (1 << 24), "%s: Hq=%d heads of %d: too wide", what, Hq, dh);
    const int64_t most = std::max(s->tiles[2], s->tiles[5]);
    CAPDEC_REQUIRE(most * Hq < (1ll << 31), "%s: too many tiles for one launch", what);
    return 0;
}

// items of one part of the table
static const PackedItem* items_of(const capdec_packed_seqs* s, int part) {
    const PackedItem* t = (const PackedItem*)s->table;
    for (int i = 0; i < part; ++i) t += s->tiles[i];
    return t;
}

#define CAPDEC_PACKED(kernel, part, heads, threads)                                                                    \
    do {                                                                                                               \
        p.items = items_of(s, part);                                                                                   \
        hipLaunchKernelGGL(kernel, dim3((unsigned)(s->tiles[part] * (heads))), dim3(threads), 0, st, p);               \
    } while (0)

// One wave a tile where most sequences fit 32 rows: a taller tile would be half empty, and its waves would wait for each
// other (200 captions of 8 to 40 tokens, 8 heads of 64, bf16: forward 6.1 us against 8.8, backward 16 / 27, fp32 50 / 84; 64
// sequences of 33 to 64, 16 heads of 128 over 4, the other way: 13 / 15, 32 / 51).
static bool short_rows(const int* tiles) { return 2 * (int64_t)tiles[2] < 3 * (int64_t)tiles[1]; }

// 128 rows a workgroup where that makes five for every four of the 256 CUs (6 prompts, 16 heads of 128: forward 157 us
// against 210 with 64 rows; 32 paragraphs, 8 heads of 128: 11.6 / 15.3, backward 37 / 43); 64 rows and two waves a block where it
// does not (10 texts of 300 to 500 tokens, 8 heads of 64, 280 tall tiles: backward 25 / 27; one text of 2000, 256: 141 / 145).
// fp32: always the latter: 32 keys of fp32 already fill the LDS of a 64-key tile, and at 128 dims 128 rows spill (32
// paragraphs 26 / 39, 8 texts 152 / 300).
template <typename T>
static bool tall_rows(const int* tiles, int heads) { return sizeof(T) == 2 && (int64_t)tiles[0] * heads >= 320; }

// bf16: 32 rows and four waves for them, each taking every fourth run of keys, where 64 rows would leave CUs without a workgroup
// (one text of 1655 tokens, 8 heads of 64: forward 21 -> 16 us, backward 44 -> 39; one of 1302, 8 heads of 128 over 4: 25 -> 24,
// 67 -> 63; with 368 tiles of 64 rows, 4 texts of 734, 8 heads of 128 over 1, the other way: 18 / 30, 65 / 78)
static bool low_rows(const int* tiles, int heads) { return (int64_t)tiles[1] * heads < 256; }

// bytes of what dq leaves for dk / dv, whole 16-byte pieces
template <typename T>
static size_t stat_bytes(int Hq, size_t stat_rows) {
    return sizeof(T) == 4 ? (Hq * stat_rows * 4 + 15) & ~(size_t)15 : Hq * stat_rows * 16;
}

// dk, dv of key tiles whose walk over the queries is longer than 5/4 of a workgroup's even share (512 run at once) are summed in
// parts by several workgroups and joined in a second launch: such a walk would be running alone at the end (8 texts of 300 to
// 4096 tokens, 16 heads of 128 over 4: 340 us in one piece, 242 and 13 for the join in parts; one text of 2000 over 2 heads,
// the whole backward: 333 / 138).  With 3/4, 1/2, 1/4 of a share the first one's backward takes 4, 8 and 23 % more.  A part is
// at least 8 tiles (4: 64 sequences of 64 to 128 tokens 33 -> 46 us, the join not being worth it).
struct PackedParts {
    int parts, items, slots;  // of the longest tiles; tiles that are split, their parts together
};
static PackedParts packed_parts(const capdec_packed_seqs* s, int Hkv, int group) {
    PackedParts c = {1, 0, 0};
    const int64_t longest = (int64_t)s->walk_max * group, all = s->walk_sum * group * Hkv;
    while (c.parts < (1 << WALK_LEVELS) && 4 * longest * 512 > 5 * all * c.parts && longest >= 16 * c.parts) c.parts *= 2;
    for (int l = 0; l < WALK_LEVELS && (c.parts >> l) > 1; ++l) {
        c.items += s->walk_levels[l];
        c.slots += s->walk_levels[l] * (c.parts >> l);
    }
    return c;
}

template <typename T, int DH>
static void launch_fwd(PackedParams& p, const capdec_packed_seqs* s, hipStream_t st) {
    if (s->one_block) CAPDEC_PACKED((packed_fwd_kernel<T, DH, 1, 1, 1, true>), 2, p.Hq, 64);
    else if (short_rows(s->tiles)) CAPDEC_PACKED((packed_fwd_kernel<T, DH, 1, 1, 1>), 2, p.Hq, 64);
    else if (sizeof(T) == 2 && low_rows(s->tiles, p.Hq)) {
        if constexpr (sizeof(T) == 2) CAPDEC_PACKED((packed_fwd_kernel<T, DH, 1, 4, 1>), 2, p.Hq, 256);
    } else if (!tall_rows<T>(s->tiles, p.Hq)) CAPDEC_PACKED((packed_fwd_kernel<T, DH, 2, 2, 1>), 1, p.Hq, 256);
    else if constexpr (sizeof(T) == 2) CAPDEC_PACKED((packed16_fwd_kernel<DH>), 0, p.Hq, 256);
}

template <typename T, int DH>
static void launch_bwd(PackedParams& p, const capdec_packed_seqs* s, hipStream_t st) {
    if (s->one_block) {
        constexpr int W = sizeof(T) == 4 && DH == 128 ? 2 : 4;
        if (s->tiles[5] == 0) return;
        if (p.group == 1) CAPDEC_PACKED((packed_bwd_block_kernel<T, DH, 1>), 5, p.Hkv, 64);
        else CAPDEC_PACKED((packed_bwd_block_kernel<T, DH, W>), 5, p.Hkv, 64 * W);
        return;
    }
    const bool one = short_rows(s->tiles + 3);
    if (sizeof(T) == 2 && !one) p.stats = p.delta;
    if (s->tiles[0] > 0) {
        if (short_rows(s->tiles)) CAPDEC_PACKED((packed_bwd_dq_kernel<T, DH, 1, 1, 1>), 2, p.Hq, 64);
        else if (sizeof(T) == 2 && low_rows(s->tiles, p.Hq)) {
            if constexpr (sizeof(T) == 2) CAPDEC_PACKED((packed_bwd_dq_kernel<T, DH, 1, 4, 1>), 2, p.Hq, 256);
        } else if (!tall_rows<T>(s->tiles, p.Hq)) CAPDEC_PACKED((packed_bwd_dq_kernel<T, DH, 2, 2, 1>), 1, p.Hq, 256);
        else if constexpr (sizeof(T) == 2) CAPDEC_PACKED((packed16_bwd_dq_kernel<DH>), 0, p.Hq, 256);
    }
    if (s->tiles[3] > 0) {
        if (one) CAPDEC_PACKED((packed_bwd_dkv_kernel<T, DH, 1, 1>), 5, p.Hkv, 64);
        else {
            const PackedParts cut = packed_parts(s, p.Hkv, p.group);
            p.parts = cut.parts;
            p.slots = cut.slots;
            for (int l = 0; l < WALK_LEVELS; ++l) p.levels[l] = s->walk_levels[l];
            p.part = (float*)((char*)p.delta + stat_bytes<T>(p.Hq, p.stat_rows));
            p.items = items_of(s, 4);
            const dim3 grid((unsigned)((s->tiles[4] - cut.items + cut.slots) * p.Hkv));
            if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((packed_bwd_dkv_kernel<T, DH, 2, 2>), grid, dim3(256), 0, st, p);
            else hipLaunchKernelGGL((packed16_bwd_dkv_kernel<DH>), grid, dim3(256), 0, st, p);
            if (cut.parts > 1) hipLaunchKernelGGL((packed_join_kernel<T, DH>), dim3((unsigned)(cut.items * p.Hkv)), dim3(256), 0, st, p);
        }
    }
}

}  // namespace capdec

// [delta or statistics][partial sums]
extern "C" size_t capdec_attn_packed_scratch_bytes(const capdec_packed_seqs* seqs, size_t stat_rows, int Hq, int Hkv, int dh, int dtype) {
    if (packed_check("capdec_attn_packed_scratch_bytes", seqs, Hq, Hkv, dh, dtype, 1.f) || seqs->one_block) return 0;
    size_t bytes = dtype == CAPDEC_F32 ? stat_bytes<float>(Hq, stat_rows) : stat_bytes<__bf16>(Hq, stat_rows);
    if (!short_rows(seqs->tiles + 3)) bytes += (size_t)packed_parts(seqs, Hkv, Hq / Hkv).slots * Hkv * 2 * 64 * dh * 4;
    return bytes;
}

extern "C" int capdec_attn_packed_fwd(const capdec_packed_seqs* seqs, const void* q, int ldq, const void* k, int ldk, const void* v,
                                      int ldv, void* o, int ldo, void* lse, size_t stat_rows, int Hq, int Hkv, int dh, int dtype,
                                      float scale, capdec_stream_t stream) {
    if (int rc = packed_check("capdec_attn_packed_fwd", seqs, Hq, Hkv, dh, dtype, scale)) return rc;
    const int es = dtype == CAPDEC_F32 ? 4 : 2;
    CAPDEC_REQUIRE(packed_mat(q, ldq, Hq * dh, es, seqs->rows_q) && packed_mat(k, ldk, Hkv * dh, es, seqs->rows_k) &&
                       packed_mat(v, ldv, Hkv * dh, es, seqs->rows_k) && packed_mat(o, ldo, Hq * dh, es, seqs->rows_q),
                   "capdec_attn_packed_fwd: matrices must be non-null, 16-byte aligned, with row strides that are multiples of 16 "
                   "bytes, cover the heads and do not pass 2^25 bytes");
    CAPDEC_REQUIRE(!lse || stat_rows >= (size_t)seqs->rows_q, "capdec_attn_packed_fwd: stat_rows=%zu below the %d query rows", stat_rows, seqs->rows_q);
    if (seqs->rows_q == 0) return 0;
    PackedParams p;
    memset(&p, 0, sizeof(p));
    p.q = q; p.k = k; p.v = v; p.out = o; p.lse = (float*)lse;
    p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
    p.Hq = Hq; p.Hkv = Hkv; p.group = Hq / Hkv; p.causal = seqs->causal; p.stat_rows = stat_rows; p.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == CAPDEC_F32) {
        if (dh == 64) launch_fwd<float, 64>(p, seqs, st);
        else launch_fwd<float, 128>(p, seqs, st);
    } else {
        if (dh == 64) launch_fwd<__bf16, 64>(p, seqs, st);
        else launch_fwd<__bf16, 128>(p, seqs, st);
    }
    return check_launch("capdec_attn_packed_fwd");
}

extern "C" int capdec_attn_packed_bwd(const capdec_packed_seqs* seqs, const void* q, int ldq, const void* k, int ldk, const void* v,
                                      int ldv, const void* o, int ldo, const void* dout, int lddo, const void* lse,
                                      size_t stat_rows, void* scratch, size_t scratch_bytes, void* dq, int lddq, void* dk, int lddk, void* dv, int lddv, int Hq, int Hkv,
                                      int dh, int dtype, float scale, capdec_stream_t stream) {
    if (int rc = packed_check("capdec_attn_packed_bwd", seqs, Hq, Hkv, dh, dtype, scale)) return rc;
    const int es = dtype == CAPDEC_F32 ? 4 : 2;
    CAPDEC_REQUIRE(packed_mat(q, ldq, Hq * dh, es, seqs->rows_q) && packed_mat(k, ldk, Hkv * dh, es, seqs->rows_k) &&
                       packed_mat(v, ldv, Hkv * dh, es, seqs->rows_k) && packed_mat(o, ldo, Hq * dh, es, seqs->rows_q) &&
                       packed_mat(dout, lddo, Hq * dh, es, seqs->rows_q) && packed_mat(dq, lddq, Hq * dh, es, seqs->rows_q) &&
                       packed_mat(dk, lddk, Hkv * dh, es, seqs->rows_k) && packed_mat(dv, lddv, Hkv * dh, es, seqs->rows_k),
                   "capdec_attn_packed_bwd: matrices must be non-null, 16-byte aligned, with row strides that are multiples of 16 "
                   "bytes, cover the heads and do not pass 2^25 bytes");
    CAPDEC_REQUIRE(seqs->rows_q == 0 || (lse && stat_rows >= (size_t)seqs->rows_q),
                   "capdec_attn_packed_bwd: lse missing, or stat_rows=%zu below the %d query rows", stat_rows, seqs->rows_q);
    const size_t need = capdec_attn_packed_scratch_bytes(seqs, stat_rows, Hq, Hkv, dh, dtype);
    CAPDEC_REQUIRE(need == 0 || (scratch && aligned16(scratch)), "capdec_attn_packed_bwd: scratch missing or not 16-byte aligned");
    if (scratch_bytes < need) {
        set_error("capdec_attn_packed_bwd: scratch of %zu bytes, %zu needed", scratch_bytes, need);
        return CAPDEC_ERR_WORKSPACE;
    }
    PackedParams p;
    memset(&p, 0, sizeof(p));
    p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = (float*)lse; p.delta = (float*)scratch;
    p.dq = dq; p.dk = dk; p.dv = dv;
    p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.lddo = lddo; p.lddq = lddq; p.lddk = lddk; p.lddv = lddv;
    p.Hq = Hq; p.Hkv = Hkv; p.group = Hq / Hkv; p.causal = seqs->causal; p.stat_rows = stat_rows; p.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == CAPDEC_F32) {
        if (dh == 64) launch_bwd<float, 64>(p, seqs, st);
        else launch_bwd<float, 128>(p, seqs, st);
    } else {
        if (dh == 64) launch_bwd<__bf16, 64>(p, seqs, st);
        else launch_bwd<__bf16, 128>(p, seqs, st);
    }
    return check_launch("capdec_attn_packed_bwd");
}
