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
// workgroup searches for its sequence and the tail of a launch is made of its shortest tiles.  Everything a row sums up
// stays inside one workgroup: no atomics, bitwise reproducible.  The backward runs twice over the scores (dq by query
// tiles, dk / dv by key tiles and all heads of the group): 7 products instead of 5, in exchange for no fp32 gradient
// block in memory and no order that depends on the launch.
#include <algorithm>
#include <new>
#include <vector>

#include "attention_tile.h"

namespace capdec {

struct PackedItem {  // one tile of rows of one sequence
    int q0, nq, k0, nk;  // the sequence's rows in the packed matrices
    int t0;              // first row of this tile within its side
    int reserved[3];
};

struct PackedParams {
    const void* q; const void* k; const void* v; const void* o; const void* dout;
    void* out; void* dq; void* dk; void* dv;
    float* lse; float* delta;
    const PackedItem* items;
    int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    int Hq, Hkv, group, causal;
    size_t stat_rows;  // rows of one head in lse / delta
    float scale;
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

template <typename T, int DH, int NW, int KB>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 2 : 1) void packed_fwd_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int BN = 32 * KB, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const T* qg = (const T*)p.q + (size_t)w.q0 * p.ldq + head * DH;
    const T* kg = (const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const T* vg = (const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + (tid >> 6) * 32;        // this wave's first row
    const int row = r0 + l31, off = w.nk - w.nq;  // causal: row sees keys j <= row + off
    const int kmax = p.causal ? min(w.nk, min(w.t0 + NW * 32, w.nq) + off) : w.nk;  // of the workgroup's last row
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    // keys the wave's rows can see at all, and keys that all of them see (no mask below)
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;

    typename L::frag qf[L::NF];
    L::load_row(qf, qg + (size_t)row * p.ldq, row < w.nq, half);
    Staged<T, DH, NW * 64, BN> ks, vs;
    if (nt > 0) {
        ks.load(kg, p.ldk, 0, w.nk, tid);
        vs.load(vg, p.ldv, 0, w.nk, tid);
        ks.store(smem, tid);
        vs.store(smem + IMG, tid);
    }
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    Running run;
    run.init();
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const unsigned char* Ks = smem + (t & 1) * 2 * IMG;
        const unsigned char* Vs = Ks + IMG;
        const bool more = t + 1 < nt;
        if (more) {
            ks.load(kg, p.ldk, (t + 1) * BN, w.nk, tid);
            vs.load(vg, p.ldv, (t + 1) * BN, w.nk, tid);
        }
        __builtin_amdgcn_sched_barrier(0);
        const int k0 = t * BN;
        if (k0 < wave_end) {
            f32x16 s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                zero16(s[b]);
                L::mma_rows(s[b], Ks + b * 32 * L::ROWB, ln, qf);  // S^T[key][query]
            }
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
                L::mma_cols(acc, Vs + b * 32 * L::ROWB, ln, pw);  // O^T[dim][query] += V^T P^T
            }
        }
        if (more) {
            unsigned char* nx = smem + ((t + 1) & 1) * 2 * IMG;
            ks.store(nx, tid);
            vs.store(nx + IMG, tid);
            __syncthreads();
        }
    }
    const float l = run.l + __shfl_xor(run.l, 32, 64);
    if (row < w.nq) {
        const bool any = run.m2 != -INFINITY || l != 0.f;  // (a NaN row is not an empty one)
        L::store_row((T*)p.out + (size_t)(w.q0 + row) * p.ldo + head * DH, acc, any ? 1.f / l : 0.f, half);
        if (p.lse && half == 0)
            p.lse[(size_t)head * p.stat_rows + w.q0 + row] = any ? (run.base() + __log2f(l)) * LN2 : -INFINITY;
    }
}

// dq and delta = rowsum(do * o); the wave owns 32 query rows
template <typename T, int DH, int NW, int KB>
__global__ __launch_bounds__(NW * 64, NW == 4 && sizeof(T) == 2 ? 2 : 1) void packed_bwd_dq_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int BN = 32 * KB, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int head, it;
    packed_place(p.Hq, head, it);
    const PackedItem w = p.items[it];
    const int hk = head / p.group;
    const T* kg = (const T*)p.k + (size_t)w.k0 * p.ldk + hk * DH;
    const T* vg = (const T*)p.v + (size_t)w.k0 * p.ldv + hk * DH;
    const int r0 = w.t0 + (tid >> 6) * 32;
    const int row = r0 + l31, off = w.nk - w.nq;
    const int kmax = p.causal ? min(w.nk, min(w.t0 + NW * 32, w.nq) + off) : w.nk;
    const int nt = kmax > 0 ? (kmax + BN - 1) / BN : 0;
    const int wave_end = r0 >= w.nq ? 0 : (p.causal ? min(w.nk, min(r0 + 32, w.nq) + off) : w.nk);
    const int all_see = p.causal ? min(w.nk, r0 + 1 + off) : w.nk;
    const bool mine = row < w.nq;
    const size_t grow = (size_t)(w.q0 + row);

    typename L::frag qf[L::NF], df[L::NF];
    float dsum;
    {
        typename L::frag of[L::NF];
        L::load_row(of, (const T*)p.o + grow * p.ldo + head * DH, mine, half);
        L::load_row(df, (const T*)p.dout + grow * p.lddo + head * DH, mine, half);
        dsum = L::dot(df, of);
        dsum += __shfl_xor(dsum, 32, 64);
    }
    L::load_row(qf, (const T*)p.q + grow * p.ldq + head * DH, mine, half);
    // p = exp2(s c - lse2); a row that sees nothing has lse = -inf: its weights are zeros
    float lse2 = mine ? p.lse[(size_t)head * p.stat_rows + grow] * LOG2E : INFINITY;
    if (lse2 == -INFINITY) lse2 = INFINITY;
    if (mine && half == 0) p.delta[(size_t)head * p.stat_rows + grow] = dsum;
    Staged<T, DH, NW * 64, BN> ks, vs;
    if (nt > 0) {
        ks.load(kg, p.ldk, 0, w.nk, tid);
        vs.load(vg, p.ldv, 0, w.nk, tid);
        ks.store(smem, tid);
        vs.store(smem + IMG, tid);
    }
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 acc[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const unsigned char* Ks = smem + (t & 1) * 2 * IMG;
        const unsigned char* Vs = Ks + IMG;
        const bool more = t + 1 < nt;
        if (more) {
            ks.load(kg, p.ldk, (t + 1) * BN, w.nk, tid);
            vs.load(vg, p.ldv, (t + 1) * BN, w.nk, tid);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int k0 = t * BN + 32 * b;
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
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = exp2_fast(__fmaf_rn(s[r], c, -lse2)) * (dp[r] - dsum);
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
    if (mine) L::store_row((T*)p.dq + grow * p.lddq + head * DH, acc, p.scale, half);
}

// dk, dv: the wave owns 32 key rows of one key / value head and walks the query tiles of every query head of the group.
// Runs after packed_bwd_dq_kernel (reads delta).
template <typename T, int DH, int NW>
__global__ __launch_bounds__(NW * 64, NW == 4 && sizeof(T) == 2 && DH == 64 ? 2 : 1) void packed_bwd_dkv_kernel(PackedParams p) {
    using L = AttTile<T, DH>;
    constexpr int BN = 32, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    __shared__ float stat[2][2][BN];  // [buffer][lse2 | delta][query]
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    int hk, it;
    packed_place(p.Hkv, hk, it);
    const PackedItem w = p.items[it];
    const int r0 = w.t0 + (tid >> 6) * 32;
    const int key = r0 + l31, off = w.nk - w.nq;
    const bool mine = key < w.nk;
    // causal: query i sees key j iff i >= j - off; the first tile that meets one of the workgroup's keys
    const int first = p.causal ? max(0, w.t0 - off) / BN : 0;
    const int per = max(0, (w.nq + BN - 1) / BN - first), nt = per * p.group;

    typename L::frag kf[L::NF], vf[L::NF];
    L::load_row(kf, (const T*)p.k + (size_t)(w.k0 + key) * p.ldk + hk * DH, mine, half);
    L::load_row(vf, (const T*)p.v + (size_t)(w.k0 + key) * p.ldv + hk * DH, mine, half);
    Staged<T, DH, NW * 64, BN> qs, ds;
    float st = 0.f;  // threads 0..31: a row's lse2, 32..63: its delta
    auto fetch = [&](int t) {
        const int head = hk * p.group + t / per, q0 = (first + t % per) * BN;
        qs.load((const T*)p.q + (size_t)w.q0 * p.ldq + head * DH, p.ldq, q0, w.nq, tid);
        ds.load((const T*)p.dout + (size_t)w.q0 * p.lddo + head * DH, p.lddo, q0, w.nq, tid);
        if (tid < 64) {
            const int i = q0 + (tid & 31);
            const float none = tid < 32 ? INFINITY : 0.f;
            const float* src = tid < 32 ? p.lse : p.delta;
            st = i < w.nq ? src[(size_t)head * p.stat_rows + w.q0 + i] : none;
            if (tid < 32) {
                st *= LOG2E;
                if (st == -INFINITY) st = INFINITY;
            }
        }
    };
    auto put = [&](int b) {
        qs.store(smem + b * 2 * IMG, tid);
        ds.store(smem + b * 2 * IMG + IMG, tid);
        if (tid < 64) stat[b][tid >> 5][tid & 31] = st;
    };
    if (nt > 0) {
        fetch(0);
        put(0);
    }
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    f32x16 dk[L::NDT], dv[L::NDT];
#pragma unroll
    for (int dt = 0; dt < L::NDT; ++dt) {
        zero16(dk[dt]);
        zero16(dv[dt]);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const unsigned char* Qs = smem + (t & 1) * 2 * IMG;
        const unsigned char* Ds = Qs + IMG;
        const bool more = t + 1 < nt;
        if (more) fetch(t + 1);
        __builtin_amdgcn_sched_barrier(0);
        const int q0 = (first + t % per) * BN;
        if (r0 < w.nk && (!p.causal || r0 <= q0 + BN - 1 + off)) {
            f32x16 s, dp;
            zero16(s);
            zero16(dp);
            L::mma_rows(s, Qs, ln, kf);   // S[query][key]
            L::mma_rows(dp, Ds, ln, vf);  // dP[query][key]
            // queries past the end have lse2 = +inf (weight zero); keys past the end are nobody's
            if (p.causal && q0 + off < r0 + 31) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = key <= q0 + row_of(r, half) + off ? s[r] : -INFINITY;
            }
            float x[16], y[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4t ls = *reinterpret_cast<const f32x4t*>(&stat[t & 1][0][8 * i + 4 * half]);
                const f32x4t de = *reinterpret_cast<const f32x4t*>(&stat[t & 1][1][8 * i + 4 * half]);
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
        if (more) {
            put((t + 1) & 1);
            __syncthreads();
        }
    }
    if (mine) {
        L::store_row((T*)p.dk + (size_t)(w.k0 + key) * p.lddk + hk * DH, dk, p.scale, half);
        L::store_row((T*)p.dv + (size_t)(w.k0 + key) * p.lddv + hk * DH, dv, 1.f, half);
    }
}

// rows per workgroup: four waves of 32, or one
constexpr int TALL = 128, SHORT = 32;

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
    return sum < (1ll << 31);
}

}  // namespace capdec

using namespace capdec;

extern "C" size_t capdec_packed_table_bytes(const int* lens_q, const int* lens_k, int n) {
    if (!lens_q || n <= 0 || !lengths_ok(lens_q, n) || (lens_k && !lengths_ok(lens_k, n))) return 0;
    const int* lk = lens_k ? lens_k : lens_q;
    const int64_t items = tiles_of(lens_q, n, TALL) + tiles_of(lens_q, n, SHORT) + tiles_of(lk, n, TALL) + tiles_of(lk, n, SHORT);
    return (size_t)(items > 0 ? items : 1) * sizeof(PackedItem);
}

extern "C" int capdec_packed_plan(const int* lens_q, const int* lens_k, int n, int causal, void* table_dev, size_t table_bytes,
                                  capdec_packed_seqs* seqs) {
    CAPDEC_REQUIRE(lens_q && table_dev && seqs && n > 0, "capdec_packed_plan: bad arguments (n=%d)", n);
    const size_t need = capdec_packed_table_bytes(lens_q, lens_k, n);
    CAPDEC_REQUIRE(need > 0, "capdec_packed_plan: a length is negative, or the rows pass 2^31");
    CAPDEC_REQUIRE(aligned16(table_dev), "capdec_packed_plan: the table must be 16-byte aligned");
    if (table_bytes < need) {
        set_error("capdec_packed_plan: table of %zu bytes, %zu needed", table_bytes, need);
        return CAPDEC_ERR_WORKSPACE;
    }
    const int* lk = lens_k ? lens_k : lens_q;
    try {
        std::vector<PackedItem> all;
        all.reserve(need / sizeof(PackedItem));
        int count[4] = {0, 0, 0, 0};
        for (int part = 0; part < 4; ++part) {  // query tiles of 128 and 32 rows, key tiles of 128 and 32 rows
            const bool keys = part >= 2;
            const int rows = part & 1 ? SHORT : TALL;
            const size_t begin = all.size();
            int q0 = 0, k0 = 0;
            for (int i = 0; i < n; ++i) {
                const int nq = lens_q[i], nk = lk[i];
                for (int t0 = 0; t0 < (keys ? nk : nq); t0 += rows) all.push_back(PackedItem{q0, nq, k0, nk, t0, {0, 0, 0}});
                q0 += nq;
                k0 += nk;
            }
            auto cost = [&](const PackedItem& a) {  // rows of the other side that the tile walks
                if (keys) return causal ? a.nq - std::max(0, a.t0 - (a.nk - a.nq)) : a.nq;
                return causal ? std::min(a.nk, a.t0 + rows + a.nk - a.nq) : a.nk;
            };
            std::stable_sort(all.begin() + begin, all.end(), [&](const PackedItem& a, const PackedItem& b) { return cost(a) > cost(b); });
            count[part] = (int)(all.size() - begin);
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
        for (int part = 0; part < 4; ++part) seqs->tiles[part] = count[part];
        seqs->table = table_dev;
    } catch (const std::exception& e) {
        set_error("capdec_packed_plan: %s", e.what());
        return CAPDEC_ERR_ARG;
    }
    return 0;
}

namespace capdec {

static bool packed_mat(const void* p, int ld, int width, int es, int rows) {
    return rows == 0 || (p && aligned16(p) && ld >= width && ld % (16 / es) == 0);
}

static int packed_check(const char* what, const capdec_packed_seqs* s, int Hq, int Hkv, int dh, int dtype, float scale) {
    CAPDEC_REQUIRE(s && s->table, "%s: no plan", what);
    CAPDEC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "%s: Hq=%d must be a positive multiple of Hkv=%d", what, Hq, Hkv);
    CAPDEC_REQUIRE(dh == 64 || dh == 128, "%s: head dim %d not in {64,128}", what, dh);
    CAPDEC_REQUIRE(dtype == CAPDEC_F32 || dtype == CAPDEC_BF16S, "%s: dtype %d: fp32 (CAPDEC_F32) or bf16 (CAPDEC_BF16S) matrices", what, dtype);
    CAPDEC_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", what);
    CAPDEC_REQUIRE((int64_t)Hq * dh < (1 << 24), "%s: Hq=%d heads of %d: too wide", what, Hq, dh);
    const int64_t most = std::max(std::max((int64_t)s->tiles[0], (int64_t)s->tiles[1]), std::max((int64_t)s->tiles[2], (int64_t)s->tiles[3]));
    CAPDEC_REQUIRE(most * Hq < (1ll << 31), "%s: too many tiles for one launch", what);
    return 0;
}

// Four waves share the tiles they walk; one wave wastes fewer rows on short sequences.
static bool tall(int tiles_tall, int tiles_short) { return 2 * (int64_t)tiles_short >= 5 * (int64_t)tiles_tall; }

template <typename T, int DH>
static void launch_fwd(PackedParams& p, const capdec_packed_seqs* s, hipStream_t st) {
    const PackedItem* table = (const PackedItem*)s->table;
    if (tall(s->tiles[0], s->tiles[1])) {
        p.items = table;
        hipLaunchKernelGGL((packed_fwd_kernel<T, DH, 4, sizeof(T) == 2 ? 2 : 1>), dim3(s->tiles[0] * p.Hq), dim3(256), 0, st, p);
    } else {
        p.items = table + s->tiles[0];
        hipLaunchKernelGGL((packed_fwd_kernel<T, DH, 1, 1>), dim3(s->tiles[1] * p.Hq), dim3(64), 0, st, p);
    }
}

template <typename T, int DH>
static void launch_bwd(PackedParams& p, const capdec_packed_seqs* s, hipStream_t st) {
    const PackedItem* table = (const PackedItem*)s->table;
    if (s->tiles[0] > 0) {
        if (tall(s->tiles[0], s->tiles[1])) {
            p.items = table;
            hipLaunchKernelGGL((packed_bwd_dq_kernel<T, DH, 4, sizeof(T) == 2 ? 2 : 1>), dim3(s->tiles[0] * p.Hq), dim3(256), 0, st, p);
        } else {
            p.items = table + s->tiles[0];
            hipLaunchKernelGGL((packed_bwd_dq_kernel<T, DH, 1, 1>), dim3(s->tiles[1] * p.Hq), dim3(64), 0, st, p);
        }
    }
    if (s->tiles[2] > 0) {
        const PackedItem* keys = table + s->tiles[0] + s->tiles[1];
        if (tall(s->tiles[2], s->tiles[3])) {
            p.items = keys;
            hipLaunchKernelGGL((packed_bwd_dkv_kernel<T, DH, 4>), dim3(s->tiles[2] * p.Hkv), dim3(256), 0, st, p);
        } else {
            p.items = keys + s->tiles[2];
            hipLaunchKernelGGL((packed_bwd_dkv_kernel<T, DH, 1>), dim3(s->tiles[3] * p.Hkv), dim3(64), 0, st, p);
        }
    }
}

}  // namespace capdec

extern "C" int capdec_attn_packed_fwd(const capdec_packed_seqs* seqs, const void* q, int ldq, const void* k, int ldk, const void* v,
                                      int ldv, void* o, int ldo, void* lse, size_t stat_rows, int Hq, int Hkv, int dh, int dtype,
                                      float scale, capdec_stream_t stream) {
    if (int rc = packed_check("capdec_attn_packed_fwd", seqs, Hq, Hkv, dh, dtype, scale)) return rc;
    const int es = dtype == CAPDEC_F32 ? 4 : 2;
    CAPDEC_REQUIRE(packed_mat(q, ldq, Hq * dh, es, seqs->rows_q) && packed_mat(k, ldk, Hkv * dh, es, seqs->rows_k) &&
                       packed_mat(v, ldv, Hkv * dh, es, seqs->rows_k) && packed_mat(o, ldo, Hq * dh, es, seqs->rows_q),
                   "capdec_attn_packed_fwd: matrices must be non-null, 16-byte aligned, with row strides that are multiples of 16 "
                   "bytes and cover the heads");
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
                                      int ldv, const void* o, int ldo, const void* dout, int lddo, const void* lse, void* delta,
                                      size_t stat_rows, void* dq, int lddq, void* dk, int lddk, void* dv, int lddv, int Hq, int Hkv,
                                      int dh, int dtype, float scale, capdec_stream_t stream) {
    if (int rc = packed_check("capdec_attn_packed_bwd", seqs, Hq, Hkv, dh, dtype, scale)) return rc;
    const int es = dtype == CAPDEC_F32 ? 4 : 2;
    CAPDEC_REQUIRE(packed_mat(q, ldq, Hq * dh, es, seqs->rows_q) && packed_mat(k, ldk, Hkv * dh, es, seqs->rows_k) &&
                       packed_mat(v, ldv, Hkv * dh, es, seqs->rows_k) && packed_mat(o, ldo, Hq * dh, es, seqs->rows_q) &&
                       packed_mat(dout, lddo, Hq * dh, es, seqs->rows_q) && packed_mat(dq, lddq, Hq * dh, es, seqs->rows_q) &&
                       packed_mat(dk, lddk, Hkv * dh, es, seqs->rows_k) && packed_mat(dv, lddv, Hkv * dh, es, seqs->rows_k),
                   "capdec_attn_packed_bwd: matrices must be non-null, 16-byte aligned, with row strides that are multiples of 16 "
                   "bytes and cover the heads");
    CAPDEC_REQUIRE(seqs->rows_q == 0 || (lse && delta && stat_rows >= (size_t)seqs->rows_q),
                   "capdec_attn_packed_bwd: lse / delta missing, or stat_rows=%zu below the %d query rows", stat_rows, seqs->rows_q);
    PackedParams p;
    memset(&p, 0, sizeof(p));
    p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = (float*)lse; p.delta = (float*)delta;
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
