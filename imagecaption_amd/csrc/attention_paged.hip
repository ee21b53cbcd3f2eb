// Attention of new tokens over a paged cache.  See include/capdec.h (capdec_attn_paged).
//
// The rows of a (sequence, key / value head) are its new tokens times the query heads of the group: they all read the same
// keys, so they share a tile.  Two kernels, both over (sequence, key / value head, split of the keys, tile of rows):
//   paged_keys_kernel  few rows (decode steps, drafted tokens): bound by the cache's bytes.  A tile of 32 or 64 rows, kept in
//                      LDS; each of the four waves streams every fourth run of 32 keys: the keys go from registers straight to
//                      the matrix instructions, the values through an LDS image of the wave's own, no barrier in the loop; the
//                      waves join at the end.
//   paged_rows_kernel  many rows (chunks of a prompt): bound by the matrix products.  A tile of 128 rows, 32 a wave, in
//                      registers; 64 keys and values at a time are shared by the waves through LDS.
// e4m3 codes become bf16 (exactly) in registers; a key's scale multiplies its scores, a value's scale its weights.
// Splits leave (maximum, sum, unnormalised context) in fp32 and a second launch joins them; a sequence short enough for one
// split writes its result at once.
#include <algorithm>

#include "attention_tile.h"
#include "paged.h"

namespace capdec {

static __device__ unsigned int g_bad_pages;
static __device__ uint4 g_zero_row[16];  // stands in for the rows of positions that do not exist

constexpr int WINDOW = 512;       // pages whose offsets are in LDS at a time
constexpr int SPLIT_MIN = 512;    // fewest keys worth a split of their own (and a second launch)
constexpr int SPLIT_WANT = 512;   // workgroups to aim at: two for each of the 256 CUs, which is what they hold

struct PagedParams {
    const void* k; const void* v; const float* ks; const float* vs;
    const __bf16* q; __bf16* o; float* lse;
    const int* cu; const int* lens; const int* table;
    float* part_o; float2* part_ml; int* part_n;
    int ldq, ldo, ld_table, cols, n, rows, Hq, Hkv, group, page_log2, pages;
    int splits, tiles, clear;
    float scale;
};

// what a workgroup works on
struct PagedItem {
    int seq, hk, split, tile, step;  // tiles tile, tile + step, ..
    int a, nq, len, kbegin, kend, nsplit;  // rows a .. a + nq - 1; keys kbegin .. kend - 1 of len
    bool ok;
};

// Keys of a split: the batch's work -- keys times tiles of rows -- shared out over SPLIT_WANT workgroups, less what the sequences'
// shorter last splits are expected to add: all of them run at once and take about as long (a prompt chunk over four sequences:
// 105 us; without that allowance 113, with the longest chunk's tiles for every chunk 126; 8 contexts of 9 to 60 thousand tokens
// with 384 / 512 / 640 workgroups to aim at: 47 / 45 / 59).  At least SPLIT_MIN keys, at least
// what the longest possible sequence needs to have no more than `splits`, in whole runs of 128.
// (In fp32: the share only has to be the same for all workgroups and, for the grid to hold all splits, no less than the work
// of a SPLIT_WANT-th, which half a tile's allowance or 2^-18 makes sure of.)
__device__ __forceinline__ int split_size(const PagedParams& p, float work, int tiles, int len) {
    const float room = fmaxf((float)SPLIT_WANT - (float)tiles * (float)p.Hkv * 0.5f, (float)SPLIT_WANT / 4);
    const float share = work * (float)p.Hkv * (1.f + 0x1p-18f) / room;
    const int c = max((int)fminf(share, 0x1p30f) + 1, (len + p.splits - 1) / p.splits);
    return (max(c, SPLIT_MIN) + 127) & ~127;
}

// sums of v over the lanes up to this one
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
#define CAPDEC_SCAN(ctrl, rows) v += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, false))
    CAPDEC_SCAN(0x111, 0xf);  // row_shr:1, 2, 4, 8: within rows of 16 lanes
    CAPDEC_SCAN(0x112, 0xf);
    CAPDEC_SCAN(0x114, 0xf);
    CAPDEC_SCAN(0x118, 0xf);
    CAPDEC_SCAN(0x142, 0xa);  // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
    CAPDEC_SCAN(0x143, 0xc);
#undef CAPDEC_SCAN
    return v;
}
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }

// Workgroup -> (sequence, split, tile of BLOCK rows), key / value head.  With splits, only as many workgroups are launched as
// there can be in all, and which one a workgroup is follows from the lengths, by a scan over them that every wave makes for
// itself.  (One workgroup for every split that the longest possible sequence could have, most of them without work: 49 us
// instead of 46 for 8 contexts of 9 to 60 thousand tokens, 29 instead of 21 for chunks of 5 drafted tokens over 48 contexts; the
// scan by the whole workgroup, through LDS: 1.4 us more.)  The row tiles of one (sequence, head, split) go round the XCDs
// (blockIdx % 8): kept on one XCD they would share its L2, but a few such groups of up to 16 tiles do not divide by eight (a
// prompt chunk over four sequences: 134 us against 123).
template <int BLOCK>
__device__ __forceinline__ PagedItem paged_place(const PagedParams& p) {
    const int tid = threadIdx.x, lane = tid & 63, cap = p.cols << p.page_log2;
    PagedItem w;
    w.split = 0;
    w.nsplit = 1;
    w.kbegin = 0;
    w.ok = true;
    int from, to, len;
    if (p.splits == 1) {
        const int pair = blockIdx.x / p.tiles;
        w.tile = blockIdx.x % p.tiles;
        w.step = p.tiles;
        w.hk = pair % p.Hkv;
        w.seq = pair / p.Hkv;
        from = p.cu ? p.cu[w.seq] : w.seq;
        to = p.cu ? p.cu[w.seq + 1] : w.seq + 1;
        len = p.lens[w.seq];
        w.len = w.kend = min(max(len, 0), cap);
    } else {
        w.hk = blockIdx.x % p.Hkv;
        const int unit = blockIdx.x / p.Hkv;
        // a lane's sequence: all three numbers are asked for at once
        auto ask = [&](int i, int& f, int& t, int& l) {
            f = i < p.n ? (p.cu ? p.cu[i] : i) : 0;
            t = i < p.n ? (p.cu ? p.cu[i + 1] : i + 1) : 0;
            l = i < p.n ? p.lens[i] : 0;
        };
        auto tiles_of = [&](int f, int t) {
            f = min(max(f, 0), p.rows);
            return max(1, ((min(max(t, f), p.rows) - f) * p.group + BLOCK - 1) / BLOCK);
        };
        int f, t, l;
        ask(lane, f, t, l);
        int tiles = lane < p.n ? tiles_of(f, t) : 0;
        float work = (float)tiles * (float)min(max(l, 0), cap);
        for (int i = lane + 64; i < p.n; i += 64) {
            int f2, t2, l2;
            ask(i, f2, t2, l2);
            const int more = tiles_of(f2, t2);
            tiles += more;
            work += (float)more * (float)min(max(l2, 0), cap);
        }
        tiles = last_lane(wave_scan(tiles));
        work = __int_as_float(last_lane(__float_as_int(wave_scan(work))));
        w.ok = false;
        int before = 0;  // workgroups (of one head) of the sequences already passed
        for (int i0 = 0; i0 < p.n; i0 += 64) {
            if (i0) ask(i0 + lane, f, t, l);
            const int kept = min(max(l, 0), cap), height = tiles_of(f, t);
            // (a length and a share together may pass 2^31)
            auto cuts = [&](int of) { return max(1, (int)(((unsigned)kept + (unsigned)of - 1u) / (unsigned)of)); };
            int size = split_size(p, work, tiles, kept), n = cuts(size);
            size = max((int)(((unsigned)kept + (unsigned)n - 1u) / (unsigned)n + 127u) & ~127, 128);  // all alike, not whole ones and a rest
            n = cuts(size);
            const int mine = i0 + lane < p.n ? n * height : 0, upto = wave_scan(mine);
            const unsigned at = (unsigned)(unit - (before + upto - mine));
            const unsigned long long own = __ballot(at < (unsigned)mine);
            if (own) {
                const int src = __ffsll(own) - 1;
                auto take = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
                const int index = take((int)at), cut = take(size);
                w.ok = true;
                w.seq = i0 + src;
                w.step = take(height);
                w.nsplit = take(n);
                w.split = min((int)((unsigned)index / (unsigned)w.step), w.nsplit - 1);
                w.tile = (int)((unsigned)index % (unsigned)w.step);
                from = take(f);
                to = take(t);
                len = take(l);
                w.len = min(max(len, 0), cap);
                w.kbegin = w.split * cut;
                w.kend = min(w.len, w.kbegin + cut);
                break;
            }
            before += last_lane(upto);
        }
        if (!w.ok) return w;
    }
    w.a = min(max(from, 0), p.rows);
    w.nq = min(max(to, w.a), p.rows) - w.a;
    if (len > cap && w.split == 0 && w.tile == 0 && w.hk == 0 && tid == 0) atomicAdd(&g_bad_pages, 1u);
    return w;
}

// rows that belong to no sequence, behind the last and before the first: zeros, if the caller wants them
template <int DH>
__device__ __forceinline__ void clear_rest(const PagedParams& p, int tid) {
    if (!p.clear) return;
    const int begin = p.cu ? min(max(p.cu[0], 0), p.rows) : 0, end = p.cu ? min(max(p.cu[p.n], begin), p.rows) : p.n;
    auto zero = [&](int row) {
        for (int i = tid; i < p.Hq * DH / 8; i += 256) reinterpret_cast<uint4*>(p.o + (size_t)row * p.ldo)[i] = uint4{0, 0, 0, 0};
    };
    for (int64_t row = blockIdx.x; row < begin; row += gridDim.x) zero((int)row);
    for (int64_t row = (int64_t)end + blockIdx.x; row < p.rows; row += gridDim.x) zero((int)row);
}

// end of the window of pages that begins at key k0: whole pages, and a multiple of 128 keys from k0 unless it is kend
__device__ __forceinline__ int window_end(const PagedParams& p, int k0, int kend) {
    const int64_t e = ((int64_t)(k0 >> p.page_log2) + WINDOW) << p.page_log2;
    return (int)min(e, (int64_t)kend);
}

// the pages of the keys k0 .. kend - 1 (one window) into LDS, as byte offsets of this head's first row there; pages outside the
// cache become -1 and are counted where `last` is set, for the chunk's last tile of rows: it sees all keys, the first one of a long
// chunk may see none of a split's or a window's.  *bad tells that there are some.  The caller waits for the workgroup before it
// uses them.
__device__ __forceinline__ void load_pages(int64_t* pages, int* bad, const PagedParams& p, const PagedItem& w, bool last, int k0, int kend, int row_bytes,
                                           int tid, int nt) {
    __syncthreads();  // the window before is no longer read
    if (tid == 0) *bad = 0;
    __syncthreads();
    const int first = k0 >> p.page_log2, n = kend > k0 ? ((kend - 1) >> p.page_log2) - first + 1 : 0;
    const int* row = p.table + (size_t)w.seq * p.ld_table + first;
    for (int i = tid; i < n; i += nt) {
        const int id = row[i];
        int64_t at = -1;
        if (id >= 0 && id < p.pages) at = (((int64_t)id * p.Hkv + w.hk) << p.page_log2) * row_bytes;
        else {
            *bad = 1;
            if (w.hk == 0 && last) atomicAdd(&g_bad_pages, 1u);
        }
        pages[i] = at;
    }
}

// No branches below: positions that do not exist are read from a row of zeros.  With branches the compiler cannot count the
// requests in flight and waits for all of them where it needs the oldest.  kend - 1 has to be a position of the split.
__device__ __forceinline__ const unsigned char* row_or_zeros(const void* base, size_t at, bool there) {
    return there ? (const unsigned char*)base + at : reinterpret_cast<const unsigned char*>(g_zero_row);
}

// ROWS keys (K) and values of one head on their way pages -> registers -> LDS images, shared out over NT threads in 16-byte
// pieces
template <bool E4M3, int DH, int NT, int ROWS, bool K>
struct PageStage {
    using L = AttTile<__bf16, DH>;
    static constexpr int RB = E4M3 ? DH : 2 * DH, PP = RB / 16, N = ROWS * PP / NT;
    static_assert(ROWS * PP % NT == 0, "every thread moves the same number of pieces");
    uint4 k[K ? N : 1], v[N];
    __device__ __forceinline__ void load(const PagedParams& p, const int64_t* pages, int first_page, int key0, int kend, int tid) {
        const int mask = (1 << p.page_log2) - 1;
        const unsigned char *ka[N], *va[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int key = key0 + (j * NT + tid) / PP, piece = (j * NT + tid) % PP;
            const int64_t page = pages[(min(key, kend - 1) >> p.page_log2) - first_page];
            const size_t at = (size_t)page + (unsigned)((key & mask) * RB + piece * 16);
            const bool there = key < kend && page >= 0;
            if constexpr (K) ka[j] = row_or_zeros(p.k, at, there);
            va[j] = row_or_zeros(p.v, at, there);
        }
        if constexpr (K) {
#pragma unroll
            for (int j = 0; j < N; ++j) k[j] = *reinterpret_cast<const uint4*>(ka[j]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = *reinterpret_cast<const uint4*>(va[j]);
    }
    __device__ static __forceinline__ void put(unsigned char* img, const uint4* r, int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int row = (j * NT + tid) / PP, piece = (j * NT + tid) % PP;
            unsigned char* at = img + row * L::ROWB;
            if constexpr (E4M3) {
                *reinterpret_cast<bf16x8p*>(at + (((2 * piece) ^ L::swz(row)) << 4)) = e4m3_to_bf16(r[j].x, r[j].y);
                *reinterpret_cast<bf16x8p*>(at + (((2 * piece + 1) ^ L::swz(row)) << 4)) = e4m3_to_bf16(r[j].z, r[j].w);
            } else {
                *reinterpret_cast<uint4*>(at + ((piece ^ L::swz(row)) << 4)) = r[j];
            }
        }
    }
};

// 32 keys of one head straight into matrix operands: a lane holds every second 16-byte piece of its key's row (its partner
// lane ^ 32 the others).  The order in which a product takes the head dimension is free as long as both operands agree:
// an e4m3 piece feeds two k-steps, so the queries' pieces are taken in that order.
template <bool E4M3, int DH>
struct KeyFrags {
    using L = AttTile<__bf16, DH>;
    static constexpr int RB = E4M3 ? DH : 2 * DH, N = RB / 32;
    uint4 r[N];
    float sk, sv;
    __device__ __forceinline__ void load(const PagedParams& p, const int64_t* pages, int first_page, int key, int kend, int half) {
        const int64_t page = pages[(min(key, kend - 1) >> p.page_log2) - first_page];
        const int at = key & ((1 << p.page_log2) - 1);
        const bool there = key < kend && page >= 0;
        const unsigned char* row = row_or_zeros(p.k, (size_t)page + (unsigned)(at * RB), there) + 16 * half;
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const uint4*>(row + (there ? 32 * i : 0));
        if constexpr (E4M3) {
            sk = *(there ? p.ks + (size_t)page / DH + at : reinterpret_cast<const float*>(g_zero_row));
            sv = *(there ? p.vs + (size_t)page / DH + at : reinterpret_cast<const float*>(g_zero_row));
        }
    }
    // acc[key][row] += keys x rows^T; q: this lane's row in the image of rows, sw: its swizzle
    __device__ __forceinline__ void mma(f32x16& acc, const unsigned char* q, int sw, int half) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (E4M3) {
                const int piece = 2 * (2 * i + half);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8t, e4m3_to_bf16(r[i].x, r[i].y)),
                                                              *reinterpret_cast<const bf16x8t*>(q + ((piece ^ sw) << 4)), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8t, e4m3_to_bf16(r[i].z, r[i].w)),
                                                              *reinterpret_cast<const bf16x8t*>(q + (((piece + 1) ^ sw) << 4)), acc, 0, 0, 0);
            } else {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8t, r[i]),
                                                              *reinterpret_cast<const bf16x8t*>(q + (((2 * i + half) ^ sw) << 4)), acc, 0, 0, 0);
            }
        }
    }
};

// scales of one key and its value; zero past the split's end or on a bad page (no branches, as above)
template <int DH>
__device__ __forceinline__ void key_scales(const PagedParams& p, const int64_t* pages, int first_page, int key, int kend, float& sk, float& sv) {
    const int64_t page = pages[(min(key, kend - 1) >> p.page_log2) - first_page];
    const size_t at = (size_t)page / DH + (key & ((1 << p.page_log2) - 1));
    const bool there = key < kend && page >= 0;
    sk = *(there ? p.ks + at : reinterpret_cast<const float*>(g_zero_row));
    sv = *(there ? p.vs + at : reinterpret_cast<const float*>(g_zero_row));
}

// scores of 32 keys from k0 on that this lane's row does not see, that lie past the split or on a bad page: -infinity
__device__ __forceinline__ void hide(f32x16& s, const PagedParams& p, const int64_t* pages, int first_page, int k0, int end, bool good, int half) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int key = k0 + row_of(r, half);
        bool there = key < end;
        if (!good && there) there = pages[(key >> p.page_log2) - first_page] >= 0;
        s[r] = there ? s[r] : -INFINITY;
    }
}

// (Weights keep 16 bits: bound by the cache's bytes, the kernel has room for the products of their second terms.  8 contexts of 9
// to 60 thousand tokens: 46 us either way; 48 of 100 to 8000, five tokens each: 21 -> 22.7.)
// R blocks of 32 rows; every wave walks its own runs of 32 keys, the next run asked for before this one's products.  The rows are
// the same for all waves and stay in LDS; values pass through an LDS image (their operand is transposed), keys go to the matrix
// instructions as they come: less LDS for a workgroup and a shorter way through each run, which is what bounds the kernel (a
// run's steps depend on each other, so the rate is the number of waves a CU holds).
// An e4m3 run stays in registers until its turn.  The values of a bf16 run do not: PageStage's array of uint4 is copied whole, and
// this compiler keeps it in private memory (160 bytes a lane at 128 dims, 96 at 64), so the wave waits for the next run's values,
// and for its keys before them, as soon as it has asked for them, and the values move three times.
template <bool E4M3, int DH, int R>
__global__ __launch_bounds__(256, DH == 128 ? (R == 1 ? 2 : 1) : (R == 1 ? 3 : 2)) void paged_keys_kernel(PagedParams p) {
    using L = AttTile<__bf16, DH>;
    constexpr int IMG = 32 * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[(4 + R) * IMG];
    __shared__ int64_t pages[WINDOW];
    __shared__ int s_bad;
    __shared__ __attribute__((aligned(16))) float sc[4][2][32];
    __shared__ float ml[4][2][32];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const PagedItem w = paged_place<32 * R>(p);
    clear_rest<DH>(p, tid);
    if (!w.ok) return;
    const int nrows = w.nq * p.group;
    constexpr int NQ = 32 * R * L::PPR / 256;
    uint4 rows[NQ];
    auto load_rows = [&](int tile) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int rl = (j * 256 + tid) / L::PPR, piece = (j * 256 + tid) % L::PPR, r = tile * 32 * R + rl;
            rows[j] = uint4{0, 0, 0, 0};
            if (r < nrows)
                rows[j] = *reinterpret_cast<const uint4*>(p.q + (size_t)(w.a + r / p.group) * p.ldq + (w.hk * p.group + r % p.group) * DH + piece * 8);
        }
    };
    load_rows(w.tile);  // (on their way while the page table is read)
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    unsigned char* Vs = smem + wave * IMG;
    unsigned char* Qs = smem + 4 * IMG;

    for (int tile = w.tile; tile * 32 * R < nrows; tile += w.step) {
        if (tile != w.tile) load_rows(tile);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int rl = (j * 256 + tid) / L::PPR, piece = (j * 256 + tid) % L::PPR;
            *reinterpret_cast<uint4*>(Qs + rl * L::ROWB + ((piece ^ L::swz(rl & 31)) << 4)) = rows[j];
        }
        int see[R];
#pragma unroll
        for (int b = 0; b < R; ++b) see[b] = min(w.kend, w.len - w.nq + (tile * 32 * R + b * 32 + l31) / p.group + 1);
        const int all_see = min(w.kend, w.len - w.nq + tile * 32 * R / p.group + 1);
        f32x16 acc[R][L::NDT];
        Running run[R];
#pragma unroll
        for (int b = 0; b < R; ++b) {
            run[b].init();
#pragma unroll
            for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[b][dt]);
        }
        for (int win = w.kbegin, wend; win < w.kend; win = wend) {
            wend = window_end(p, win, w.kend);
            load_pages(pages, &s_bad, p, w, (tile + 1) * 32 * R >= nrows, win, wend, E4M3 ? DH : 2 * DH, tid, 256);
            __syncthreads();  // pages, rows
            const bool good = s_bad == 0;
            const int first_page = win >> p.page_log2;
            KeyFrags<E4M3, DH> kf;
            PageStage<E4M3, DH, 64, 32, false> st;
            int k0 = win + wave * 32;
            if (k0 < wend) {
                kf.load(p, pages, first_page, k0 + l31, wend, half);
                st.load(p, pages, first_page, k0, wend, lane);
            }
            for (; k0 < wend; k0 += 128) {
                f32x16 s[R];
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    zero16(s[b]);
                    kf.mma(s[b], Qs + b * IMG + l31 * L::ROWB, L::swz(l31), half);  // S^T[key][row]
                }
                // one wave's LDS operations execute in order: the previous run's reads are done before these writes land
                if (E4M3 && half == 0) {
                    sc[wave][0][l31] = kf.sk;
                    sc[wave][1][l31] = kf.sv;
                }
                st.put(Vs, st.v, lane);
                if (k0 + 128 < wend) {
                    kf.load(p, pages, first_page, k0 + 128 + l31, wend, half);
                    st.load(p, pages, first_page, k0 + 128, wend, lane);
                }
                wave_fence();
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    if constexpr (E4M3) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const f32x4t f = *reinterpret_cast<const f32x4t*>(&sc[wave][0][8 * i + 4 * half]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) s[b][4 * i + j] *= f[j];
                        }
                    }
                    if (!good || k0 + 32 > all_see) hide(s[b], p, pages, first_page, k0, see[b], good, half);
                    float top = s[b][0];
#pragma unroll
                    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[b][r]);
                    bool raised;
                    const float a = run[b].raise(top, c, &raised);
                    if (raised) {
#pragma unroll
                        for (int dt = 0; dt < L::NDT; ++dt)
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[b][dt][r] *= a;
                    }
                    const float base = run[b].base();
                    float x[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4t f = {1.f, 1.f, 1.f, 1.f};
                        if constexpr (E4M3) f = *reinterpret_cast<const f32x4t*>(&sc[wave][1][8 * i + 4 * half]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float e = exp2_fast(__fmaf_rn(s[b][4 * i + j], c, -base));
                            run[b].l += e;
                            x[4 * i + j] = E4M3 ? e * f[j] : e;
                        }
                    }
                    typename L::weights2 pw;
                    L::pack(pw, x);
                    L::mma_cols(acc[b], Vs, ln, pw);
                }
                wave_fence();
            }
        }
        // join the four waves: statistics first, then the contexts, half the dims at a time, through their (now free) images
#pragma unroll
        for (int b = 0; b < R; ++b) {
            const float l = run[b].l + __shfl_xor(run[b].l, 32, 64);
            if (half == 0) {
                ml[wave][0][l31] = run[b].m2;
                ml[wave][1][l31] = l;
            }
            __syncthreads();
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, ml[i][0][l31]);
            const float mine = run[b].m2 == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(run[b].m2 - m);
            const int rl = tid >> 3, r = tile * 32 * R + b * 32 + rl;  // eight threads a row
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) mm = fmaxf(mm, ml[i][0][rl]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float mi = ml[i][0][rl], li = ml[i][1][rl];
                ll += mi == -INFINITY ? li : li * exp2_fast(mi - mm);
            }
            const int token = r / p.group, head = w.hk * p.group + r % p.group, grow = w.a + token;
            const bool any = ll != 0.f;
            const size_t at = (size_t)grow * p.Hq + head;
            const float inv = any ? 1.f / ll : 0.f;
            constexpr int HD = DH / 2, PIECES = HD / 4;  // dims of a half, 16-byte pieces of an fp32 row of them
            float* ctx = reinterpret_cast<float*>(Vs);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h) __syncthreads();
#pragma unroll
                for (int dt = h * L::NDT / 2; dt < (h + 1) * L::NDT / 2; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int piece = (dt - h * L::NDT / 2) * 8 + 2 * i + half;
                        const f32x4t v = {acc[b][dt][4 * i] * mine, acc[b][dt][4 * i + 1] * mine, acc[b][dt][4 * i + 2] * mine,
                                          acc[b][dt][4 * i + 3] * mine};
                        *reinterpret_cast<f32x4t*>(ctx + l31 * HD + ((piece ^ (l31 & 7)) << 2)) = v;
                    }
                __syncthreads();
                if (r < nrows) {
#pragma unroll
                    for (int j = 0; j < PIECES / 8; ++j) {
                        const int piece = j * 8 + (tid & 7);
                        f32x4t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            v += *reinterpret_cast<const f32x4t*>(reinterpret_cast<const float*>(smem + i * IMG) + rl * HD + ((piece ^ (rl & 7)) << 2));
                        if (w.nsplit == 1) {
                            const bf16x4t out = {(__bf16)(v[0] * inv), (__bf16)(v[1] * inv), (__bf16)(v[2] * inv), (__bf16)(v[3] * inv)};
                            *reinterpret_cast<bf16x4t*>(p.o + (size_t)grow * p.ldo + head * DH + h * HD + piece * 4) = out;
                        } else {
                            *reinterpret_cast<f32x4t*>(p.part_o + ((size_t)w.split * p.rows * p.Hq + at) * DH + h * HD + piece * 4) = v;
                        }
                    }
                }
            }
            if (r < nrows && (tid & 7) == 0) {
                if (w.nsplit == 1) {
                    if (p.lse) p.lse[(size_t)head * p.rows + grow] = any ? ((mm == -INFINITY ? 0.f : mm) + __log2f(ll)) * LN2 : -INFINITY;
                } else {
                    p.part_ml[(size_t)w.split * p.rows * p.Hq + at] = float2{mm, ll};
                }
                if (w.split == 0 && p.part_n) p.part_n[at] = w.nsplit;
            }
            __syncthreads();
        }
    }
}

// 128 rows, 32 a wave; 64 keys at a time shared by the waves.  bf16 pages travel by DMA one tile ahead; e4m3 pages pass
// through registers, where they become bf16.  (At 128 dims a wave is at its 256 registers: two are spilled for bf16 pages, four
// for e4m3; they are stored before the walk over the keys and taken back behind it.)
template <bool E4M3, int DH>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedParams p) {
    using L = AttTile<__bf16, DH>;
    constexpr int KB = 2, BN = 32 * KB, IMG = BN * L::ROWB;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * IMG];
    __shared__ int64_t pages[WINDOW];
    __shared__ int s_bad;
    __shared__ __attribute__((aligned(16))) float sc[2][2][BN];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const PagedItem w = paged_place<128>(p);
    clear_rest<DH>(p, tid);
    if (!w.ok) return;
    const int nrows = w.nq * p.group;
    const typename L::lanes ln = L::make_lanes(lane);
    const float c = p.scale * LOG2E;
    for (int tile = w.tile; tile * 128 < nrows; tile += w.step) {
        const int r0 = tile * 128 + wave * 32, r = r0 + l31, token = r / p.group, head = w.hk * p.group + r % p.group;
        const int see = min(w.kend, w.len - w.nq + token + 1);
        const int all_see = min(w.kend, w.len - w.nq + r0 / p.group + 1);
        const int wave_end = r0 < nrows ? min(w.kend, w.len - w.nq + min(r0 + 31, nrows - 1) / p.group + 1) : 0;
        const int end = min(w.kend, w.len - w.nq + min(tile * 128 + 127, nrows - 1) / p.group + 1);
        typename L::frag qf[L::NF];
        L::load_row(qf, p.q + (size_t)(w.a + token) * p.ldq + head * DH, r < nrows, half);
        f32x16 acc[L::NDT];
#pragma unroll
        for (int dt = 0; dt < L::NDT; ++dt) zero16(acc[dt]);
        Running run;
        run.init();
        landed(qf);
        for (int win = w.kbegin, wend; win < end; win = wend) {
            wend = window_end(p, win, w.kend);
            load_pages(pages, &s_bad, p, w, (tile + 1) * 128 >= nrows, win, wend, E4M3 ? DH : 2 * DH, tid, 256);  // (the images are free from here on, too)
            __syncthreads();
            const bool good = s_bad == 0;
            const int first_page = win >> p.page_log2, nt = (min(end, wend) - win + BN - 1) / BN;
            PageStage<E4M3, DH, 256, BN, true> st;
            float sk, sv;
            // tile t into the images at img: by DMA at once, or into registers (put stores them)
            auto fetch = [&](int t, unsigned char* img) {
                const int k0 = win + t * BN;
                if constexpr (E4M3) {
                    st.load(p, pages, first_page, k0, wend, tid);
                    if (tid < BN) key_scales<DH>(p, pages, first_page, k0 + tid, wend, sk, sv);
                } else {
                    constexpr int PER = 64 / L::PPR, N = BN / PER / 4;  // rows of a 1 KiB transfer, transfers of a wave
                    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(
                        (int)(unsigned)(size_t)(const __attribute__((address_space(3))) unsigned char*)(img + wave * N * 1024));
                    const int mask = (1 << p.page_log2) - 1;
                    int64_t at[N];
                    unsigned within[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const int rl = (wave * N + j) * PER + lane / L::PPR, key = min(k0 + rl, wend - 1);
                        at[j] = pages[(key >> p.page_log2) - first_page];
                        within[j] = (unsigned)((key & mask) * L::ROWB) + (((unsigned)(lane % L::PPR)) ^ (unsigned)L::swz(rl & 31)) * 16u;
                    }
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const unsigned char* ka = (const unsigned char*)p.k + at[j] + within[j];
                        const unsigned char* va = (const unsigned char*)p.v + at[j] + within[j];
                        if (!good && at[j] < 0) ka = va = reinterpret_cast<const unsigned char*>(g_zero_row) + within[j] % L::ROWB;
                        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to + j * 1024), "v"(ka) : "memory");
                        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to + IMG + j * 1024), "v"(va) : "memory");
                    }
                }
            };
            auto put = [&](int t, unsigned char* img) {
                if constexpr (E4M3) {
                    st.put(img, st.k, tid);
                    st.put(img + IMG, st.v, tid);
                    if (tid < BN) {
                        sc[t & 1][0][tid] = sk;
                        sc[t & 1][1][tid] = sv;
                    }
                }
            };
            auto turn = [&](int t, unsigned char* cur, unsigned char* nx) __attribute__((always_inline)) {
                const unsigned char* Ks = cur;
                const unsigned char* Vs = Ks + IMG;
                const bool more = t + 1 < nt;
                if constexpr (!E4M3) dma_sync();
                if (more) fetch(t + 1, nx);
                __builtin_amdgcn_sched_barrier(0);
                const int k0 = win + t * BN;
                if (k0 < wave_end) {
                    f32x16 s[KB];
                    bf16x8t kf[KB][L::NF], vf[2 * L::NDT];
#pragma unroll
                    for (int b = 0; b < KB; ++b) L::read_rows(kf[b], Ks + b * 32 * L::ROWB, ln);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int b = 0; b < KB; ++b) zero16(s[b]);
#pragma unroll
                    for (int ks = 0; ks < L::NF; ++ks)
#pragma unroll
                        for (int b = 0; b < KB; ++b) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[b][ks], qf[ks], s[b], 0, 0, 0);  // S^T[key][row]
                    L::read_cols(vf, Vs, ln);
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (E4M3) {
#pragma unroll
                        for (int b = 0; b < KB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const f32x4t f = *reinterpret_cast<const f32x4t*>(&sc[t & 1][0][32 * b + 8 * i + 4 * half]);
#pragma unroll
                                for (int j = 0; j < 4; ++j) s[b][4 * i + j] *= f[j];
                            }
                    }
                    if (!good || k0 + BN > all_see) {
#pragma unroll
                        for (int b = 0; b < KB; ++b) hide(s[b], p, pages, first_page, k0 + 32 * b, see, good, half);
                    }
                    float top = s[0][0];
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
                    bool raised;
                    const float a = run.raise(top, c, &raised);
                    if (raised) {
#pragma unroll
                        for (int dt = 0; dt < L::NDT; ++dt)
#pragma unroll
                            for (int i = 0; i < 16; ++i) acc[dt][i] *= a;
                    }
                    const float base = run.base();
#pragma unroll
                    for (int b = 0; b < KB; ++b) {
                        float x[16];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            f32x4t f = {1.f, 1.f, 1.f, 1.f};
                            if constexpr (E4M3) f = *reinterpret_cast<const f32x4t*>(&sc[t & 1][1][32 * b + 8 * i + 4 * half]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float e = exp2_fast(__fmaf_rn(s[b][4 * i + j], c, -base));
                                run.l += e;
                                x[4 * i + j] = E4M3 ? e * f[j] : e;
                            }
                        }
                        typename L::weights pw;
                        L::pack(pw, x);
                        L::mma_read_cols(acc, vf, pw);  // O^T[dim][row] += V^T P^T
                        if (b + 1 < KB) L::read_cols(vf, Vs + (b + 1) * 32 * L::ROWB, ln);
                    }
                }
                if constexpr (E4M3) {
                    if (more) {
                        put(t + 1, nx);
                        __syncthreads();
                    }
                }
            };
            fetch(0, smem);
            put(0, smem);
            if constexpr (E4M3) __syncthreads();
            for (int t = 0; t < nt; t += 2) {
                turn(t, smem, smem + 2 * IMG);
                if (t + 1 < nt) turn(t + 1, smem + 2 * IMG, smem);
            }
        }
        const float l = run.l + __shfl_xor(run.l, 32, 64);
        if (r < nrows) {
            const int grow = w.a + token;
            const bool any = l != 0.f;
            const size_t at = (size_t)grow * p.Hq + head;
            if (w.nsplit == 1) {
                L::store_row(p.o + (size_t)grow * p.ldo + head * DH, acc, any ? 1.f / l : 0.f, half);
                if (p.lse && half == 0) p.lse[(size_t)head * p.rows + grow] = any ? (run.base() + __log2f(l)) * LN2 : -INFINITY;
            } else {
                const size_t sat = (size_t)w.split * p.rows * p.Hq + at;
                AttTile<float, DH>::store_row(p.part_o + sat * DH, acc, 1.f, half);
                if (half == 0) p.part_ml[sat] = float2{run.m2, l};
            }
            if (half == 0 && w.split == 0 && p.part_n) p.part_n[at] = w.nsplit;
        }
    }
}

// The splits' contexts of one (row, head) by W waves that take every W-th split and join in wave order: four where there
// are few rows, one where there are many.
template <int DH, int W>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
    __shared__ float box[4][DH + 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = wave % W;
    const size_t all = (size_t)p.rows * p.Hq, at = (size_t)blockIdx.x * (4 / W) + wave / W;
    const int grow = (int)(at / p.Hq), head = (int)(at % p.Hq);
    int n = 0;
    if (at < all && (p.cu ? (grow >= p.cu[0] && grow < p.cu[p.n]) : grow < p.n)) n = min(p.part_n[at], p.splits);
    if (n <= 1) return;  // W > 1: the whole workgroup has this item
    float m = -INFINITY;
    for (int s = lane; s < n; s += 64) m = fmaxf(m, p.part_ml[s * all + at].x);
    m = wave_max(m);
    float l = 0.f;
    constexpr int E = DH / 64;
    float acc[E] = {};
#pragma unroll 4
    for (int s = part; s < n; s += W) {
        const float2 v = p.part_ml[s * all + at];
        const float f = v.x == -INFINITY ? (v.y == 0.f ? 0.f : 1.f) : exp2_fast(v.x - m);
        l += v.y * f;
        const float* src = p.part_o + (s * all + at) * DH + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __fmaf_rn(src[e], f, acc[e]);
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) box[wave][lane * E + e] = acc[e];
        if (lane == 0) box[wave][DH] = l;
        __syncthreads();
        if (wave > 0) return;
        l = ((box[0][DH] + box[1][DH]) + box[2][DH]) + box[3][DH];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = lane * E + e;
            acc[e] = ((box[0][i] + box[1][i]) + box[2][i]) + box[3][i];
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    __bf16* dst = p.o + (size_t)grow * p.ldo + head * DH + lane * E;
    if constexpr (E == 2) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        *reinterpret_cast<pair*>(dst) = pair{(__bf16)(acc[0] * inv), (__bf16)(acc[1] * inv)};
    } else {
        dst[0] = (__bf16)(acc[0] * inv);
    }
    if (p.lse && lane == 0) p.lse[(size_t)head * p.rows + grow] = l != 0.f ? ((m == -INFINITY ? 0.f : m) + __log2f(l)) * LN2 : -INFINITY;
}

int paged_bad_count(unsigned int* count, bool reset) {
    if (hipMemcpyFromSymbol(count, HIP_SYMBOL(g_bad_pages), sizeof(unsigned int)) != hipSuccess) return CAPDEC_ERR_LAUNCH;
    if (reset && *count) {
        const unsigned int zero = 0;
        if (hipMemcpyToSymbol(HIP_SYMBOL(g_bad_pages), &zero, sizeof(zero)) != hipSuccess) return CAPDEC_ERR_LAUNCH;
    }
    return 0;
}

struct PagedShape {
    bool rows_kernel;
    int block, tiles, splits;  // rows of a tile, tiles of the longest chunk, splits of the longest sequence
    int64_t blocks;            // workgroups
};

static PagedShape paged_shape(const capdec_kv_cache* c, int n, int rows, int max_q, int Hq, int table_cols) {
    PagedShape s;
    const int64_t group = Hq / c->heads, high = max_q * group;
    s.rows_kernel = high > 64;
    s.block = s.rows_kernel ? 128 : (high > 32 ? 64 : 32);
    s.tiles = (int)((high + s.block - 1) / s.block);
    // tiles of all chunks together, at most: by their rows, with one that is not full for each
    const int64_t all = rows * group / s.block + n;
    // the longest sequence of a ragged batch gets up to four times the even share of splits
    const int64_t keys = (int64_t)table_cols * c->page, units = std::min((int64_t)n * s.tiles, all) * c->heads;
    int64_t splits = units >= SPLIT_WANT ? 1 : (4 * SPLIT_WANT + units - 1) / units;
    splits = std::min(splits, (keys + SPLIT_MIN - 1) / SPLIT_MIN);
    s.splits = (int)std::max<int64_t>(splits, 1);
    // s_i splits for t_i tiles, each of at least a share: sum s_i t_i <= sum t_i (keys_i / share + 1), and share is at least
    // sum keys_i t_i heads / SPLIT_WANT
    s.blocks = (s.splits == 1 ? (int64_t)n * s.tiles : std::min(all * s.splits, SPLIT_WANT / c->heads + 1 + all)) * c->heads;
    return s;
}

static int paged_check(const char* what, const capdec_kv_cache* c, int n, int rows, int max_q, int Hq, int table_cols) {
    if (int rc = kv_cache_check(what, c)) return rc;
    CAPDEC_REQUIRE(n > 0 && rows >= 0 && max_q > 0 && table_cols > 0, "%s: bad shape n=%d rows=%d max_q=%d table_cols=%d", what, n, rows, max_q, table_cols);
    CAPDEC_REQUIRE(Hq > 0 && Hq % c->heads == 0 && (int64_t)Hq * c->dh < (1 << 24), "%s: Hq=%d must be a multiple of the cache's %d heads", what, Hq, c->heads);
    CAPDEC_REQUIRE((int64_t)table_cols * c->page < (1ll << 31) - (1 << 20), "%s: a page table of %d columns passes 2^31 positions", what, table_cols);
    CAPDEC_REQUIRE((int64_t)rows * (Hq / c->heads) < (1ll << 30) && (int64_t)max_q * (Hq / c->heads) < (1ll << 30), "%s: too many rows", what);
    const PagedShape s = paged_shape(c, n, rows, max_q, Hq, table_cols);
    CAPDEC_REQUIRE(s.blocks < (1ll << 31) && (int64_t)rows * Hq < (1ll << 31),
                   "%s: too much work for one launch", what);
    return 0;
}

// [part_o][part_ml][part_n], each rounded up to 256 bytes
static size_t paged_bytes(int splits, int rows, int Hq, int dh, size_t* ml, size_t* cnt) {
    const size_t items = (size_t)rows * Hq;
    *ml = (splits * items * dh * 4 + 255) & ~(size_t)255;
    *cnt = *ml + ((splits * items * 8 + 255) & ~(size_t)255);
    return *cnt + items * 4;
}

}  // namespace capdec

using namespace capdec;

extern "C" size_t capdec_attn_paged_workspace_bytes(const capdec_kv_cache* cache, int n, int rows, int max_q, int Hq, int table_cols) {
    if (paged_check("capdec_attn_paged_workspace_bytes", cache, n, rows, max_q, Hq, table_cols)) return 0;
    const PagedShape s = paged_shape(cache, n, rows, max_q, Hq, table_cols);
    size_t a, b;
    return s.splits == 1 ? 0 : paged_bytes(s.splits, rows, Hq, cache->dh, &a, &b);
}

extern "C" int capdec_attn_paged(const capdec_kv_cache* cache, const void* q, int ldq, const int* cu_q, const int* kv_lens,
                                 const int* page_table, int ld_table, int table_cols, int n, int rows, int max_q, int Hq, float scale,
                                 void* o, int ldo, int clear, void* lse, void* workspace, size_t workspace_bytes, capdec_stream_t stream) {
    if (int rc = paged_check("capdec_attn_paged", cache, n, rows, max_q, Hq, table_cols)) return rc;
    CAPDEC_REQUIRE(kv_lens && page_table && ld_table >= table_cols, "capdec_attn_paged: lengths / page table missing, or ld_table=%d below %d columns",
                   ld_table, table_cols);
    CAPDEC_REQUIRE(cu_q || rows >= n, "capdec_attn_paged: %d rows for %d sequences of one token", rows, n);
    CAPDEC_REQUIRE(scale_ok(scale), "capdec_attn_paged: scale must lie between 2^-60 and 2^60");
    if (rows == 0) return 0;
    CAPDEC_REQUIRE(q && o && aligned16(q) && aligned16(o) && ldq % 8 == 0 && ldo % 8 == 0 && ldq >= Hq * cache->dh && ldo >= Hq * cache->dh,
                   "capdec_attn_paged: q / o must be non-null, 16-byte aligned bf16 matrices with row strides that are multiples of 8 and cover "
                   "the heads");
    const PagedShape s = paged_shape(cache, n, rows, max_q, Hq, table_cols);
    PagedParams p;
    memset(&p, 0, sizeof(p));
    if (s.splits > 1) {
        size_t ml, cnt;
        const size_t need = paged_bytes(s.splits, rows, Hq, cache->dh, &ml, &cnt);
        CAPDEC_REQUIRE(workspace && aligned16(workspace), "capdec_attn_paged: workspace missing or not 16-byte aligned");
        if (workspace_bytes < need) {
            set_error("capdec_attn_paged: workspace of %zu bytes, %zu needed", workspace_bytes, need);
            return CAPDEC_ERR_WORKSPACE;
        }
        p.part_o = (float*)workspace;
        p.part_ml = (float2*)((char*)workspace + ml);
        p.part_n = (int*)((char*)workspace + cnt);
    }
    p.k = cache->k; p.v = cache->v; p.ks = (const float*)cache->k_scale; p.vs = (const float*)cache->v_scale;
    p.q = (const __bf16*)q; p.o = (__bf16*)o; p.lse = (float*)lse;
    p.cu = cu_q; p.lens = kv_lens; p.table = page_table;
    p.ldq = ldq; p.ldo = ldo; p.ld_table = ld_table; p.cols = table_cols; p.n = n; p.rows = rows;
    p.Hq = Hq; p.Hkv = cache->heads; p.group = Hq / cache->heads; p.page_log2 = log2_of(cache->page); p.pages = cache->pages;
    p.splits = s.splits; p.tiles = s.tiles; p.clear = clear != 0; p.scale = scale;
    const unsigned blocks = (unsigned)s.blocks;
    const bool e = cache->dtype == CAPDEC_E4M3, wide = cache->dh == 128;
    hipStream_t st = (hipStream_t)stream;
#define CAPDEC_PAGED(E, D)                                                                                       \
    do {                                                                                                         \
        if (s.rows_kernel) hipLaunchKernelGGL((paged_rows_kernel<E, D>), dim3(blocks), dim3(256), 0, st, p);     \
        else if (s.block == 64) hipLaunchKernelGGL((paged_keys_kernel<E, D, 2>), dim3(blocks), dim3(256), 0, st, p); \
        else hipLaunchKernelGGL((paged_keys_kernel<E, D, 1>), dim3(blocks), dim3(256), 0, st, p);                \
    } while (0)
    if (e && wide) CAPDEC_PAGED(true, 128);
    else if (e) CAPDEC_PAGED(true, 64);
    else if (wide) CAPDEC_PAGED(false, 128);
    else CAPDEC_PAGED(false, 64);
#undef CAPDEC_PAGED
    if (s.splits > 1) {
        const size_t items = (size_t)rows * Hq;
        const bool few = items < 4096;
        const dim3 grid((unsigned)(few ? items : (items + 3) / 4));
        if (wide && few) hipLaunchKernelGGL((paged_join_kernel<128, 4>), grid, dim3(256), 0, st, p);
        else if (wide) hipLaunchKernelGGL((paged_join_kernel<128, 1>), grid, dim3(256), 0, st, p);
        else if (few) hipLaunchKernelGGL((paged_join_kernel<64, 4>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((paged_join_kernel<64, 1>), grid, dim3(256), 0, st, p);
    }
    return check_launch("capdec_attn_paged");
}
