// Register and LDS tiles of the packed / paged attention kernels (attention_packed.hip, attention_paged.hip).
//
// A tile is 32 rows of one head of a row-major matrix, kept in LDS as an image [32 rows][DH] whose 16-byte piece c of
// row r sits at slot c ^ swz(r).  Two products read it:
//   mma_rows   acc[image row][lane's column] += image x frag^T, reduced over the head dimension (scores: K or Q image
//              against the wave's own rows, which stay in registers as B fragments);
//   mma_cols   out[head dim][lane's column] += image^T x weights, reduced over the image's rows (context and gradients):
//              the 32 weights of a column are the accumulator of a mma_rows product, in the order in which the matrix
//              instruction left them, so probabilities never move between lanes; image rows from `rows` on have no weight.
// bf16: v_mfma_f32_32x32x16_bf16, the transposed operand comes from the transposing LDS read (ds_read_b64_tr_b16);
// fp32: v_mfma_f32_32x32x2_f32 (exact products), where any lane can read its transposed element directly.
#pragma once
#include "attention_common.h"

namespace capdec {

typedef __bf16 bf16x8t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4t __attribute__((ext_vector_type(4)));
typedef short s16x4t __attribute__((ext_vector_type(4)));
typedef float f32x4t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}

template <typename T, int DH>
struct AttTile;

template <int DH>
struct AttTile<__bf16, DH> {
    static constexpr int ES = 2, ROWB = DH * ES, PPR = ROWB / 16, EPP = 8, NF = DH / 16, NDT = DH / 32;
    typedef bf16x8t frag;  // one 16-deep k-step of a row: elements 16 ks + 8 half + 0..7
    struct weights { bf16x8t f[2]; };
    // one swizzle for both reads: 16 consecutive rows of one piece -> 16 slots (row fragments), 4 consecutive rows x 4
    // pieces -> all 64 banks (transposing reads)
    __device__ static __forceinline__ int swz(int r) {
        return DH == 128 ? (((r & 3) << 2) | ((r >> 2) & 3)) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
    }
    // lane constants of the two reads
    struct lanes {
        int row, col[2];
    };
    __device__ static __forceinline__ lanes make_lanes(int lane) {
        const int l31 = lane & 31, half = lane >> 5;
        lanes o;
        o.row = l31 * ROWB + ((half ^ swz(l31)) << 4);
        // lane 4 q + p of 16-lane group g addresses row 8 rd + 4 half + q, 8-byte piece p of the 16 columns (g & 1) * 16
        const int g4 = lane >> 4, q4 = (lane & 15) >> 2, p4 = lane & 3;
#pragma unroll
        for (int rd = 0; rd < 2; ++rd) {
            const int kr = 8 * rd + 4 * (g4 >> 1) + q4;
            o.col[rd] = kr * ROWB + ((((g4 & 1) * 2 + (p4 >> 1)) ^ swz(kr)) << 4) + 8 * (p4 & 1);
        }
        return o;
    }
    __device__ static __forceinline__ void load_row(frag* f, const __bf16* row, bool valid, int half) {
#pragma unroll
        for (int ks = 0; ks < NF; ++ks) {
            if (valid) f[ks] = *reinterpret_cast<const bf16x8t*>(row + 16 * ks + 8 * half);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) f[ks][e] = (__bf16)0.f;
        }
    }
    __device__ static __forceinline__ float dot(const frag* a, const frag* b) {
        float s = 0.f;
#pragma unroll
        for (int ks = 0; ks < NF; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __fmaf_rn((float)a[ks][e], (float)b[ks][e], s);
        return s;
    }
    __device__ static __forceinline__ void mma_rows(f32x16& acc, const unsigned char* img, const lanes& l, const frag* b) {
#pragma unroll
        for (int ks = 0; ks < NF; ++ks) {
            const bf16x8t a = *reinterpret_cast<const bf16x8t*>(img + (l.row ^ (ks << 5)));
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[ks], acc, 0, 0, 0);
        }
    }
    // the same with both operands in LDS
    __device__ static __forceinline__ void mma_images(f32x16& acc, const unsigned char* img, const unsigned char* own, const lanes& l) {
#pragma unroll
        for (int ks = 0; ks < NF; ++ks) {
            const bf16x8t a = *reinterpret_cast<const bf16x8t*>(img + (l.row ^ (ks << 5)));
            const bf16x8t b = *reinterpret_cast<const bf16x8t*>(own + (l.row ^ (ks << 5)));
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
        }
    }
    __device__ static __forceinline__ void pack(weights& w, const float* x) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < 8; ++e) w.f[m][e] = (__bf16)x[8 * m + e];
    }
    // weights that keep 16 bits: the rounded ones and what the rounding left, added by products of their own
    struct weights2 { weights hi, lo; };
    __device__ static __forceinline__ void pack(weights2& w, const float* x) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w.hi.f[m][e] = (__bf16)x[8 * m + e];
                w.lo.f[m][e] = (__bf16)(x[8 * m + e] - (float)w.hi.f[m][e]);
            }
    }
    __device__ static __forceinline__ void mma_cols(f32x16* out, const unsigned char* img, const lanes& l, const weights2& w, int rows = 32) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < NDT && 16 * m < rows; ++dt) {
                const bf16x4t lo = read_tr(img + m * 16 * ROWB + (l.col[0] ^ (dt << 6)));
                const bf16x4t hi = read_tr(img + m * 16 * ROWB + (l.col[1] ^ (dt << 6)));
                const bf16x8t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.lo.f[m], out[dt], 0, 0, 0);
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.hi.f[m], out[dt], 0, 0, 0);
            }
    }
    __device__ static __forceinline__ bf16x4t read_tr(const unsigned char* p) {
        typedef __attribute__((address_space(3))) bf16x4t lds4;
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4*)p);
    }
    __device__ static __forceinline__ void mma_cols(f32x16* out, const unsigned char* img, const lanes& l, const weights& w) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const bf16x4t lo = read_tr(img + m * 16 * ROWB + (l.col[0] ^ (dt << 6)));
                const bf16x4t hi = read_tr(img + m * 16 * ROWB + (l.col[1] ^ (dt << 6)));
                const bf16x8t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.f[m], out[dt], 0, 0, 0);
            }
    }
    // the two steps of mma_rows / mma_cols apart, for callers that read ahead
    __device__ static __forceinline__ void read_rows(bf16x8t* f, const unsigned char* img, const lanes& l) {
#pragma unroll
        for (int ks = 0; ks < NF; ++ks) f[ks] = *reinterpret_cast<const bf16x8t*>(img + (l.row ^ (ks << 5)));
    }
    __device__ static __forceinline__ void read_cols(bf16x8t* f, const unsigned char* img, const lanes& l) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const bf16x4t lo = read_tr(img + m * 16 * ROWB + (l.col[0] ^ (dt << 6)));
                const bf16x4t hi = read_tr(img + m * 16 * ROWB + (l.col[1] ^ (dt << 6)));
                f[m * NDT + dt] = bf16x8t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
    }
    __device__ static __forceinline__ void mma_read_cols(f32x16* out, const bf16x8t* a, const weights& w) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[m * NDT + dt], w.f[m], out[dt], 0, 0, 0);
    }
    // accumulators (rows = head dim, column = this lane's matrix row) -> that row, rounded once to bf16
    __device__ static __forceinline__ void store_row(__bf16* dst, const f32x16* acc, float mul, int half) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x4t v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = (__bf16)(acc[dt][4 * i + j] * mul);
                *reinterpret_cast<bf16x4t*>(dst + dt * 32 + 8 * i + 4 * half) = v;
            }
    }
};

template <int DH>
struct AttTile<float, DH> {
    static constexpr int ES = 4, ROWB = DH * ES, PPR = ROWB / 16, EPP = 4, NF = DH / 8, NDT = DH / 32;
    typedef f32x4t frag;  // elements 8 i + 4 half + 0..3: four 2-deep products take one element of each half-wave
    struct weights { float f[16]; };
    typedef weights weights2;
    struct lanes { int l31, half; };
    __device__ static __forceinline__ int swz(int r) { return r & 15; }
    __device__ static __forceinline__ lanes make_lanes(int lane) { return lanes{lane & 31, lane >> 5}; }
    __device__ static __forceinline__ void load_row(frag* f, const float* row, bool valid, int half) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            if (valid) f[i] = *reinterpret_cast<const f32x4t*>(row + 8 * i + 4 * half);
            else f[i] = f32x4t{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ static __forceinline__ float dot(const frag* a, const frag* b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __fmaf_rn(a[i][e], b[i][e], s);
        return s;
    }
    __device__ static __forceinline__ void mma_rows(f32x16& acc, const unsigned char* img, const lanes& l, const frag* b) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const f32x4t a = *reinterpret_cast<const f32x4t*>(img + l.l31 * ROWB + (((2 * i + l.half) ^ swz(l.l31)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[i][j], acc, 0, 0, 0);
        }
    }
    __device__ static __forceinline__ void mma_images(f32x16& acc, const unsigned char* img, const unsigned char* own, const lanes& l) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const int at = l.l31 * ROWB + (((2 * i + l.half) ^ swz(l.l31)) << 4);
            const f32x4t a = *reinterpret_cast<const f32x4t*>(img + at), b = *reinterpret_cast<const f32x4t*>(own + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
        }
    }
    __device__ static __forceinline__ void pack(weights& w, const float* x) {
#pragma unroll
        for (int r = 0; r < 16; ++r) w.f[r] = x[r];
    }
    __device__ static __forceinline__ void mma_cols(f32x16* out, const unsigned char* img, const lanes& l, const weights& w, int rows = 32) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (8 * (r >> 2) >= rows) continue;
            const int kr = row_of(r, l.half);
            const unsigned char* row = img + kr * ROWB + (l.l31 & 3) * 4;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const float a = *reinterpret_cast<const float*>(row + (((dt * 8 + (l.l31 >> 2)) ^ swz(kr)) << 4));
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w.f[r], out[dt], 0, 0, 0);
            }
        }
    }
    __device__ static __forceinline__ void store_row(float* dst, const f32x16* acc, float mul, int half) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4t v = {acc[dt][4 * i] * mul, acc[dt][4 * i + 1] * mul, acc[dt][4 * i + 2] * mul, acc[dt][4 * i + 3] * mul};
                *reinterpret_cast<f32x4t*>(dst + dt * 32 + 8 * i + 4 * half) = v;
            }
    }
};

// Orders a wave's LDS writes before other lanes' reads (and reads before the next writes) for the compiler; the hardware
// executes one wave's LDS operations in order, so nothing is waited for.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// a value the compiler has to take as it is here: nothing made from it is kept from an earlier turn of a loop
__device__ __forceinline__ void opaque(int& x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void opaque(unsigned& x) { asm volatile("" : "+v"(x)); }

// row fragments loaded before a loop are taken there: left to the compiler, the wait for them would stand inside the loop
// and drain the loop's own requests every turn
template <typename F, int N>
__device__ __forceinline__ void landed(F (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// lane constants made anew: the LDS addresses of a turn are not kept for the next one (fp32 has 16 of them for every 32 head
// dims; kept, they push the accumulators out of the registers)
template <int DH>
__device__ __forceinline__ void renew(typename AttTile<float, DH>::lanes& l) { opaque(l.l31); }
template <int DH>
__device__ __forceinline__ void renew(typename AttTile<__bf16, DH>::lanes&) {}

// ---- tiles that travel global -> LDS without registers (bf16) -------------------------------------------------------
template <int DH>
struct DmaTile : AttTile<__bf16, DH> {
    using B = AttTile<__bf16, DH>;
    static constexpr int ROWS_PER = 64 / B::PPR;  // rows of one 1 KiB transfer
    // Rows row0 .. row0 + ROWS - 1 of a matrix (head slice at g) -> image, shared out over NW waves; rows past the last one
    // (n - 1) are copies of it.  ROWS * ROWB / 1024 / NW transfers a wave, each from a uniform base plus a 32-bit lane
    // offset.  Inline assembly because the compiler, where it knows of a transfer in flight, waits for it before every
    // transposing LDS read (it cannot tell that the transfer fills another image); the caller waits with dma_sync.  M0 is
    // written and used here only: the compiler sets it anew before every use of its own.
    // Lane offsets: the swizzle is linear over XOR, so the row block of a transfer only flips bits of the lane's piece, and
    // its rows go into the uniform base: one vector instruction a transfer, two registers kept.
    template <int ROWS, int NW>
    struct Fetch {
        static constexpr int N = ROWS / ROWS_PER / NW;
        static_assert(ROWS % (ROWS_PER * NW) == 0, "every wave moves the same number of transfers");
        unsigned piece, row;  // byte offsets of the lane's piece in row block 0 and of its row there
        __device__ __forceinline__ void init(int ld, int lane) {
            const int r = lane / B::PPR;
            piece = (((unsigned)(lane % B::PPR)) ^ (unsigned)B::swz(r)) * 16u;
            row = (unsigned)r * ((unsigned)ld * 2u);
        }
        __device__ __forceinline__ void operator()(unsigned char* img, const __bf16* g, int ld, int row0, int n, int wave, int lane) const {
            const char* base = (const char*)(g + (size_t)row0 * ld);
            const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane(
                (int)(unsigned)(size_t)(const __attribute__((address_space(3))) unsigned char*)(img + wave * N * 1024));
            if (row0 + ROWS <= n) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int r0 = (wave * N + j) * ROWS_PER;
                    send(to + j * 1024, base + (size_t)r0 * ((unsigned)ld * 2u), (piece ^ ((unsigned)B::swz(r0) << 4)) + row);
                }
            } else {
                int own = lane / B::PPR;
                opaque(own);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int r0 = (wave * N + j) * ROWS_PER, r = min(r0 + own, n - 1 - row0);
                    send(to + j * 1024, base, (piece ^ ((unsigned)B::swz(r0) << 4)) + (unsigned)r * ((unsigned)ld * 2u));
                }
            }
        }
        __device__ static __forceinline__ void send(unsigned to, const char* base, unsigned off) {
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
        }
    };
};
// every transfer of this wave has landed, and every wave of the workgroup has come this far and has its reads of the images:
// the compiler places its own waits where a value is used, which may be behind a barrier that it does not see as one of memory
__device__ __forceinline__ void dma_sync() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// scores are scaled by any factor from 2^-60 to 2^60 (beyond, lse / scale and its like leave fp32)
static inline bool scale_ok(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }

// ROWS consecutive rows of a matrix on their way global -> registers -> LDS image, shared out over NT threads in
// 16-byte pieces.  Rows at or past `n` become zeros: a weight of zero times whatever lies behind the last row (the next
// sequence, a page's unused places) must not become NaN.
template <typename T, int DH, int NT, int ROWS>
struct Staged {
    using L = AttTile<T, DH>;
    static constexpr int N = ROWS * L::PPR / NT;
    static_assert(ROWS * L::PPR % NT == 0, "every thread moves the same number of pieces");
    uint4 r[N];
    __device__ __forceinline__ void load(const T* g, int ld, int row0, int n, int tid) {
        // uniform base plus a 32-bit lane offset; no branch between the requests of a tile that lies inside the matrix
        const char* base = (const char*)(g + (size_t)row0 * ld);
        const unsigned pitch = (unsigned)ld * (unsigned)L::ES;
        if (row0 + ROWS <= n) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned row = (j * NT + tid) / L::PPR, piece = (j * NT + tid) % L::PPR;
                r[j] = *reinterpret_cast<const uint4*>(base + (row * pitch + piece * 16u));
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned row = (j * NT + tid) / L::PPR, piece = (j * NT + tid) % L::PPR;
                r[j] = uint4{0, 0, 0, 0};
                if (row0 + (int)row < n) r[j] = *reinterpret_cast<const uint4*>(base + (row * pitch + piece * 16u));
            }
        }
    }
    __device__ __forceinline__ void store(unsigned char* img, int tid) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int row = (j * NT + tid) / L::PPR, piece = (j * NT + tid) % L::PPR;
            *reinterpret_cast<uint4*>(img + row * L::ROWB + ((piece ^ L::swz(row)) << 4)) = r[j];
        }
    }
};

// Running softmax of one column (query) whose rows (keys) arrive in blocks.  The maximum is only raised when a new score
// exceeds it by RAISE (in powers of two): weights may then reach 2^RAISE, which fp32 sums and bf16 weights hold with the
// same relative error, and the common block needs neither the exchange between the half-waves nor the rescale of the
// accumulators (64 multiplies a lane at 128 dims).
constexpr float RAISE = 8.f;
struct Running {
    float m2, l;  // reference point (scores times scale * log2 e), sum of the lane's own weights
    __device__ __forceinline__ void init() { m2 = -INFINITY; l = 0.f; }
    // top: the lane's largest raw score of the block; returns the factor the accumulators have to be scaled by (wave-uniform
    // decision: 1 for every lane when no lane needs it, and then *raised is false)
    __device__ __forceinline__ float raise(float top, float c, bool* raised) {
        const float t2 = top * c;
        *raised = __any(t2 > m2 + RAISE) != 0;
        if (!*raised) return 1.f;
        const float both = fmaxf(t2, __shfl_xor(t2, 32, 64));
        const float m_new = fmaxf(m2, both);
        const float a = m_new == -INFINITY ? 1.f : exp2_fast(m2 - m_new);
        m2 = m_new;
        l *= a;
        return a;
    }
    __device__ __forceinline__ float base() const { return m2 == -INFINITY ? 0.f : m2; }
};

}  // namespace capdec
