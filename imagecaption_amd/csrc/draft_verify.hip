// Verification of drafted tokens: accept while u q(x) < p(x), then draw from max(p - q, 0) (or from p) by inverse CDF.  See
// include/capdec.h (capdec_draft_verify).
//
// One workgroup for each sequence.  Only one row of p and one of q matter (the place of the first refusal), so the
// bytes are those two rows: the acceptance tests of all drafted tokens run on one wave's lanes at once, then 16 waves
// stream the row, each a contiguous sixteenth of it, and sum their weights in fp64 -- the sum decides which token a uniform
// hits, and fp32 sums over tens of thousands of weights would move the borders.  The wave that holds the border walks its
// part again (its bytes are in L2) with a running sum.  One launch, no workspace.
#include "common.h"

namespace capdec {

struct VerifyParams {
    const float* target; const float* draft; const int64_t* tokens; const int* num_draft; const float* u_accept; const float* u_sample;
    int64_t* out; int* accepted;
    int64_t target_seq, target_row, draft_seq, draft_row, pad;
    int ldt, ldu, drafts, V;
};

constexpr int VWAVES = 16;

__device__ __forceinline__ double shfl_up_d(double v, int o) {
    const unsigned long long b = __double_as_longlong(v);
    const unsigned lo = __shfl_up((unsigned)b, o, 64), hi = __shfl_up((unsigned)(b >> 32), o, 64);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long b = __double_as_longlong(v);
        const unsigned lo = __shfl_xor((unsigned)b, o, 64), hi = __shfl_xor((unsigned)(b >> 32), o, 64);
        v += __longlong_as_double(((unsigned long long)hi << 32) | lo);
    }
    return v;
}

// weight of one token: mode 0 = p, 1 = max(p - q, 0), 2 = p without the (sure) drafted token; NaN counts as 0
__device__ __forceinline__ double weight(float p, float q, int mode) {
    const double w = mode == 1 ? (double)p - (double)q : (double)p;
    return w > 0.0 ? w : 0.0;
}

__global__ __launch_bounds__(VWAVES * 64) void draft_verify_kernel(VerifyParams p) {
    __shared__ int s_count, s_num;
    __shared__ double part[VWAVES];
    __shared__ int s_last[VWAVES];
    __shared__ int s_pick;
    const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t* tok = p.tokens + (size_t)b * p.ldt;
    if (wave == 0) {
        // (the loads do not wait for one another: the count, then every lane its token and uniform, then the probabilities)
        const int mine = min(lane, p.drafts - 1);
        const int64_t x = p.drafts ? tok[mine] : -1;
        const float u = p.drafts ? p.u_accept[(size_t)b * p.ldu + mine] : 1.f;
        const int num = p.num_draft ? min(max(p.num_draft[b], 0), p.drafts) : p.drafts;
        bool take = false;
        if (x >= 0 && x < p.V) {
            const double pt = p.target[(size_t)b * p.target_seq + (size_t)mine * p.target_row + x];
            const double q = p.draft ? (double)p.draft[(size_t)b * p.draft_seq + (size_t)mine * p.draft_row + x] : 1.0;
            take = lane < num && (double)u * q < pt;  // exact: two 24-bit factors
        }
        const unsigned long long ok = __ballot(take);
        if (lane == 0) {
            s_count = ok == ~0ull ? 64 : __ffsll(~ok) - 1;
            s_num = num;
            s_pick = p.V;
        }
    }
    __syncthreads();
    const int count = s_count;
    const float* pr = p.target + (size_t)b * p.target_seq + (size_t)count * p.target_row;
    const float* qr = count < s_num && p.draft ? p.draft + (size_t)b * p.draft_seq + (size_t)count * p.draft_row : pr;
    int mode = count < s_num ? (p.draft ? 1 : 2) : 0;
    const int64_t sure = mode == 2 ? tok[count] : -1;  // (outside the vocabulary: removes nothing)
    // each wave a contiguous run of whole 256-element steps
    const int seg = ((p.V + VWAVES * 256 - 1) / (VWAVES * 256)) * 256;
    const int v0 = min(p.V, wave * seg), v1 = min(p.V, v0 + seg);
    const bool vec = ((reinterpret_cast<uintptr_t>(pr) | reinterpret_cast<uintptr_t>(qr)) & 15) == 0;
    auto four = [&](int v, double* w) {
        float a[4] = {0.f, 0.f, 0.f, 0.f}, c[4] = {0.f, 0.f, 0.f, 0.f};
        if (vec && v + 4 <= v1) {
            const float4 x = *reinterpret_cast<const float4*>(pr + v);
            a[0] = x.x; a[1] = x.y; a[2] = x.z; a[3] = x.w;
            if (mode == 1) {
                const float4 y = *reinterpret_cast<const float4*>(qr + v);
                c[0] = y.x; c[1] = y.y; c[2] = y.z; c[3] = y.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < v1) {
                    a[e] = pr[v + e];
                    if (mode == 1) c[e] = qr[v + e];
                }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = mode == 2 && v + e == sure ? 0.0 : weight(a[e], c[e], mode);
    };
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double sum = 0.0;
        int last = -1;
#pragma unroll 4
        for (int v = v0 + lane * 4; v < v1; v += 256) {
            double w[4];
            four(v, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum += w[e];
                if (w[e] > 0.0) last = v + e;
            }
        }
        sum = wave_sum_d(sum);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
        if (lane == 0) {
            part[wave] = sum;
            s_last[wave] = last;
        }
        __syncthreads();
        total = 0.0;
        for (int i = 0; i < VWAVES; ++i) total += part[i];
        if (total > 0.0 || mode == 0) break;
        mode = 0;  // nothing left of p - q: draw from p
        __syncthreads();
    }
    const double t = (double)p.u_sample[b] * total;
    double before = 0.0;
    for (int i = 0; i < wave; ++i) before += part[i];
    // the first wave whose running sum passes t walks its part; its border is certain to the rounding of the sums
    if (before + part[wave] > t && !(before > t)) {
        double run = before;
        bool found = false;
        for (int vv = v0; vv < v1 && !found; vv += 256) {
            const int v = vv + lane * 4;
            double w[4];
            four(v, w);
            double mine = w[0] + w[1] + w[2] + w[3], upto = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double x = shfl_up_d(upto, o);
                if (lane >= o) upto += x;
            }
            // (the scan sums each lane's part in an order of its own: a lane without weight may be the first to pass t, by a last
            // bit -- it holds no token to take)
            const unsigned long long hit = __ballot(mine > 0.0 && run + upto > t);
            if (hit) {
                found = true;
                const int first = __ffsll(hit) - 1;
                if (lane == first) {
                    double r = run + (upto - mine);
                    int pick = -1;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        r += w[e];
                        if (pick < 0 && w[e] > 0.0 && (r > t || e == 3)) pick = v + e;
                    }
                    if (pick < 0)  // rounding: the lane's last token of positive weight
                        for (int e = 3; e >= 0; --e)
                            if (pick < 0 && w[e] > 0.0) pick = v + e;
                    if (pick >= 0) atomicMin(&s_pick, pick);
                }
            }
            run += __longlong_as_double(((unsigned long long)(unsigned)__shfl((unsigned)(__double_as_longlong(upto) >> 32), 63, 64) << 32) |
                                        (unsigned)__shfl((unsigned)__double_as_longlong(upto), 63, 64));
        }
        if (!found && lane == 0) atomicMin(&s_pick, s_last[wave] >= 0 ? s_last[wave] : p.V);
    }
    __syncthreads();
    if (tid == 0) {
        int pick = s_pick;
        if (pick >= p.V) {  // no running sum passed t: the last token of positive weight, or 0
            pick = 0;
            for (int i = 0; i < VWAVES; ++i) pick = max(pick, s_last[i]);
        }
        p.out[(size_t)b * (p.drafts + 1) + count] = pick;
        p.accepted[b] = count;
    }
    if (tid <= p.drafts && tid != count) p.out[(size_t)b * (p.drafts + 1) + tid] = tid < count ? tok[tid] : p.pad;
}

}  // namespace capdec

using namespace capdec;

extern "C" int capdec_draft_verify(const void* target, int64_t target_seq, int64_t target_row, const void* draft, int64_t draft_seq,
                                   int64_t draft_row, const int64_t* tokens, int ldt, const int* num_draft, const void* u_accept, int ldu,
                                   const void* u_sample, int n, int drafts, int V, int64_t pad, int64_t* out, int* accepted,
                                   capdec_stream_t stream) {
    CAPDEC_REQUIRE(n >= 0 && drafts >= 0 && drafts <= 64 && V > 0 && V < (1 << 30), "capdec_draft_verify: bad shape n=%d drafts=%d V=%d (at most 64 drafts)",
                   n, drafts, V);
    if (n == 0) return 0;
    CAPDEC_REQUIRE(target && u_sample && out && accepted && (drafts == 0 || (tokens && u_accept && ldt >= drafts && ldu >= drafts)),
                   "capdec_draft_verify: null pointer or a row stride below %d drafts", drafts);
    CAPDEC_REQUIRE(target_row >= V && target_seq >= 0 && (!draft || (draft_row >= V && draft_seq >= 0)),
                   "capdec_draft_verify: row strides must cover the vocabulary");
    VerifyParams p;
    memset(&p, 0, sizeof(p));
    p.target = (const float*)target; p.draft = drafts ? (const float*)draft : nullptr; p.tokens = tokens; p.num_draft = num_draft;
    p.u_accept = (const float*)u_accept; p.u_sample = (const float*)u_sample; p.out = out; p.accepted = accepted;
    p.target_seq = target_seq; p.target_row = target_row; p.draft_seq = draft_seq; p.draft_row = draft_row; p.pad = pad;
    p.ldt = ldt; p.ldu = ldu; p.drafts = drafts; p.V = V;
    hipLaunchKernelGGL(draft_verify_kernel, dim3(n), dim3(VWAVES * 64), 0, (hipStream_t)stream, p);
    return check_launch("capdec_draft_verify");
}
