// Truncated categorical sampling from given uniform numbers: temperature, top-k, top-p and min-p, and the ancestral
// update of the absorbing graph built on it.  Counterpart in the reference: utils/catsample.py:10-13 (Gumbel arg-max over
// the whole vocabulary) and sampling/sampling.py:102-132 (the update that calls it); the truncations are this library's.
//
// Definition, for a row of scores x, noise u and the row's T, k, P, m (all in 64 bits; the token is that of exact
// arithmetic, not of one order of rounding):
//     q_j  = exp((x_j - max x) / T)                          entries of -inf or NaN are no candidates
//     rank = place of j by (x descending, index ascending)
//     kept = rank < k  and  sum of q ranked before j < P * (sum of q over rank < k)  and  q_j >= m;  rank 0 always
//     out  = arg max over kept of q_j / (1e-10 - log(min(u_j + 1e-10, 1)))   (u + 1e-10 rounded to 32 bits), lowest index
// q_j / E_j with E_j exponential has its maximum at j with probability q_j / sum q, so the noise picks among what is kept.
//
// No sort and no running sum: the kept entries are a PREFIX of the order.  The arg-max over everything is found first; one
// pass gives its rank and the mass before it; if it is kept, it is the answer, and if it is not, neither is anything ranked
// behind it, so the next candidate is the arg-max among what is ranked before it.  A row ends after 1/(kept mass) tries
// or about log(V / kept) of them, whichever is less, since each rejection cuts the prefix at a random place.
#include "common.h"

struct SampleArgs {
    const void* x;
    int64_t ld;
    const float* u;
    int64_t ldu;
    const float *T, *P, *m;  // per batch element, or NULL: the scalars below
    const int* k;
    float T0, P0, m0;
    int k0;
    const int64_t* xcur;  // current tokens: only rows that hold mask_id are sampled, the others keep theirs
    int64_t mask_id;
    const float* move;  // per batch element: a masked row is sampled only where u[row][V] < move
    int64_t* out;
    int64_t M, L;
    int V;
};

struct RowParams {
    float T, P, m;
    int k;
};
__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int64_t b) {
    RowParams r;
    r.T = a.T ? a.T[b] : a.T0;
    r.P = a.P ? a.P[b] : a.P0;
    r.m = a.m ? a.m[b] : a.m0;
    r.k = a.k ? a.k[b] : a.k0;
    if (r.k <= 0 || r.k > a.V) r.k = a.V;
    return r;
}
// batch element of a row (0 where no parameter goes by it): in 32 bits where the rows allow, a 64-bit division is hundreds of
// instructions
__device__ __forceinline__ int64_t batch_of_row(const SampleArgs& a, int64_t row) {
    if (!a.T && !a.P && !a.m && !a.k && !a.move) return 0;
    if (a.M < ((int64_t)1 << 31)) return a.L >= a.M ? 0 : (int64_t)((uint32_t)row / (uint32_t)a.L);
    return row / a.L;
}
// whether the row is sampled at all; otherwise its token stays
__device__ __forceinline__ bool row_moves(const SampleArgs& a, int64_t row, int64_t b) {
    if (!a.xcur) return true;
    if (a.xcur[row] != a.mask_id) return false;
    return !a.move || a.u[row * a.ldu + a.V] < a.move[b];
}
__device__ __forceinline__ int64_t row_empty(const SampleArgs& a) { return a.xcur ? a.mask_id : (int64_t)-1; }

// fp32 -> unsigned with the same order (both zeros alike); -inf and NaN: 0, no candidate
__device__ __forceinline__ uint32_t order_key(float v) {
    v += 0.0f;
    const uint32_t b = __float_as_uint(v);
    const uint32_t key = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return v > -INFINITY ? key : 0u;
}
// u + 1e-10 in 32 bits as the reference's catsample rounds it, kept inside (0, 1] whatever u is
__device__ __forceinline__ float noise_arg(float u) { return __builtin_amdgcn_fmed3f(u + 1e-10f, 1e-10f, 1.0f); }

// NT threads joined over one row in 64 bits; every member is called by all of them.  The sums inside a wave go by DPP moves: by
// shuffles, through the LDS crossbar at each of six steps, they were most of the time that a near row takes.
template <int NT> struct Joint {
    static constexpr int NW = NT / 64;
    double* sd;  // [NW] each
    int* si;
    __device__ __forceinline__ double sum(double v) {
        v = dpp_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = v;
        __syncthreads();
        v = sd[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += sd[w];
        return v;
    }
    __device__ __forceinline__ int isum(int v) {
        v = dpp_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) si[threadIdx.x >> 6] = v;
        __syncthreads();
        v = si[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += si[w];
        return v;
    }
    // largest v, lowest index among equals
    __device__ __forceinline__ void best(double& v, int& i) {
        const double top = dpp_max(v);
        i = dpp_min(v == top ? i : INT32_MAX);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { sd[threadIdx.x >> 6] = top; si[threadIdx.x >> 6] = i; }
        __syncthreads();
        v = sd[0];
        i = si[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const double ov = sd[w];
            const int oi = si[w];
            if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
        }
    }
};

// ------------------------------------------------------------------------------------------- the same in 32 bits
// Per row the 32-bit pass either settles the decision or gives the row up to resolve_row64.  What its quantities are off by
// (v_exp_f32, v_log_f32 and v_rcp_f32 measured below 2^-23 relative):
//   q_j: d2 = (x - max) * (log2 e / T) has four roundings, so q_j is off by |d2| 4 2^-24 ln 2 + 2^-23 relative.
//   q_j / E_j: a winner has q_j >= (1 / 23.1) * 1e-10, the smallest E over the largest (the first of the order has q = 1), so
//     |d2| <= 38 and the ratio is off by 7.0e-6; two of them are told apart when they differ by more than 1.4e-5: RATIO_TOL.
//   S, W: sum q |d2| <= W log2 V, so a sum is off by (log2 V * 2.8 + 2) 2^-24 W and by its n adds one after the other, n 2^-24 W:
//     V <= 64 in one lane 5.0e-6 W; 64 a lane and 10 across, V = 32768: 7.1e-6 W.  S against P W: 1.42e-5 W at most: MASS_TOL.
// Both tolerances are 1.53e-5.  A comparison nearer than that, and every row whose maximum or temperature leaves the range of
// these bounds, is "near".  Counted over normal scores: with top-p one row in 22000 to 38000 at V = 26, in 7000 to 49000 from V = 300
// on, at top-p 0.3 (the answer changes more often there) in 5000 to 24000; without top-p one in 49000 or fewer.
#define RATIO_TOL 0x1p-16f
#define MASS_TOL 0x1p-16f
#define LOG2E 1.44269504f
#define LN2 0.693147181f

__device__ __forceinline__ float inv_noise(float u) {  // 1 / E
    const float l2 = __builtin_amdgcn_logf(noise_arg(u));
    return __builtin_amdgcn_rcpf(__builtin_fmaf(-LN2, l2, 1e-10f));
}
// log2(e) / T, and whether T lies where the bounds hold
__device__ __forceinline__ float rate_of(float T, bool& near) {
    near = near || !(T > 1e-30f && T < 1e30f);
    return LOG2E / T;
}
// a number on the key scale back as the float it stands for
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}
// a key found down to bit LOW, completed: below zero the order turns the bits round, and a bf16 value's low half is all ones there
template <int LOW> __device__ __forceinline__ uint32_t whole_key(uint32_t t) {
    return t && !(t >> 31) ? t | ((1u << LOW) - 1u) : t;
}
enum Decision { KEPT, DROPPED, NEAR };
// what the 32-bit numbers say about the entry of a given rank, mass before it and weight
__device__ __forceinline__ Decision decide(const RowParams& rp, int rank, float S, float W, float q, float best, float second) {
    if (rank != 0) {
        const float margin = rp.P * W - S, tol = MASS_TOL * W;
        if (rank >= rp.k || (rp.P < 1.f && margin < -tol) || q < rp.m * (1.f - RATIO_TOL)) return DROPPED;
        if ((rp.P < 1.f && !(margin > tol)) || (rp.m > 0.f && !(q > rp.m * (1.f + RATIO_TOL)))) return NEAR;
    }
    return second < best * (1.f - RATIO_TOL) ? KEPT : NEAR;
}

// ------------------------------------------------------------------------------- the definition itself, in 64 bits
// Three forms.  A wave with an entry per lane (V <= 64): the rank of every entry and the mass before it in one loop over the
// lanes, then the arg-max over what is kept.
template <typename T> __device__ int64_t resolve_lanes64(const SampleArgs& a, int64_t row, int64_t b) {
    const int lane = threadIdx.x & 63;
    const RowParams rp = row_params(a, b);
    const float v = lane < a.V ? to_f32<T>(((const T*)a.x + row * a.ld)[lane]) + 0.0f : -INFINITY;
    const float u = lane < a.V ? (a.u + row * a.ldu)[lane] : 0.5f;
    const bool in = v > -INFINITY;
    const float mx = dpp_max(in ? v : -INFINITY);
    if (!(mx > -INFINITY)) return row_empty(a);
    if (!(rp.T > 0.f)) return __builtin_ctzll(__ballot(v == mx));  // greedy
    const double q = !in ? 0.0 : v == mx ? 1.0 : mx == INFINITY ? 0.0 : exp(((double)v - (double)mx) / (double)rp.T);
    const double r = in ? q / (1e-10 - log((double)noise_arg(u))) : -1.0;
    int rank = 0;
    double S = 0.0;
    for (int i = 0; i < a.V; ++i) {
        const float vi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
        const int lo = __builtin_amdgcn_readlane((int)__double2loint(q), i), hi = __builtin_amdgcn_readlane((int)__double2hiint(q), i);
        if ((vi > v) | ((vi == v) & (i < lane))) {  // (false for NaN)
            ++rank;
            S += __hiloint2double(hi, lo);
        }
    }
    const double W = dpp_sum(rank < rp.k ? q : 0.0);
    const bool kept = in && (rank == 0 || (rank < rp.k && (!(rp.P < 1.f) || S < (double)rp.P * W) && !(q < (double)rp.m)));
    const double best = dpp_max(kept ? r : -1.0);
    return __builtin_ctzll(__ballot(kept && r == best));
}
// A block with the row's scores, weights and ratios in LDS (V <= STAGED).  kth: what wide_row has found for the row (its t), 0 if it
// is not known (the search for it in here took more than all the rest: 20 us of 40 at V = 2365).
#define STAGED 4096
struct StagedRow {
    double q[STAGED], r[STAGED];
    float x[STAGED];
};
template <typename T, int NT>
__device__ int64_t resolve_staged64(const SampleArgs& a, int64_t row, int64_t b, uint32_t kth, StagedRow& s, double* sd, int* si) {
    Joint<NT> J{sd, si};
    const int lane = threadIdx.x & (NT - 1), V = a.V;
    const T* px = (const T*)a.x + row * a.ld;
    const float* u = a.u + row * a.ldu;
    const RowParams rp = row_params(a, b);
    const int none = INT32_MAX;
    __syncthreads();
    double top = -1.0;  // (an order key, so that one reduction serves)
    int mi = none;
    {
        // all loads at once (a thread by itself waits for each), the noise into the place of the ratios
        constexpr int NE = STAGED / NT;
        T xe[NE];
        float ue[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int j = i * NT + lane;
            xe[i] = px[j < V ? j : 0];
            ue[i] = u[j < V ? j : 0];
        }
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int j = i * NT + lane;
            const float v = to_f32<T>(xe[i]);
            const uint32_t key = j < V ? order_key(v) : 0u;
            s.x[j] = key ? v : -INFINITY;
            s.r[j] = (double)ue[i];
            if (key && (double)key > top) { top = (double)key; mi = j; }
        }
    }
    J.best(top, mi);
    if (mi == none) return row_empty(a);
    if (!(rp.T > 0.f)) return mi;  // greedy
    const float mx = s.x[mi];
    for (int j = lane; j < V; j += NT) {
        const float v = s.x[j];
        const double q = v == mx ? 1.0 : !(v > -INFINITY) || mx == INFINITY ? 0.0 : exp(((double)v - (double)mx) / (double)rp.T);
        s.q[j] = q;
        s.r[j] = v > -INFINITY ? q / (1e-10 - log((double)noise_arg((float)s.r[j]))) : -1.0;
    }
    double W = 0.0;
    if (rp.P < 1.f) {
        uint32_t t = kth;  // the k-th largest key, or 0 if there are no k candidates
        for (int bit = 31; !kth && rp.k < V && bit >= 0; --bit) {
            const uint32_t ct = t | (1u << bit);
            int n = 0;
            for (int j = lane; j < V; j += NT) n += order_key(s.x[j]) >= ct;
            n = J.isum(n);
            if (n >= rp.k) t = ct;
            if (n == rp.k) break;  // (then exactly the k first are at or above t)
        }
        double border = 0.0;
        int n = 0, any = 0;
        for (int j = lane; j < V; j += NT) {
            const uint32_t key = order_key(s.x[j]);
            if (key > t) { W += s.q[j]; ++n; }
            else if (key == t && t) border = s.q[j];
        }
        W = J.sum(W);
        if (t) {
            n = J.isum(n);
            J.best(border, any);
            W += (double)(rp.k - n) * border;  // of equal entries at the border the lowest indices are in; they weigh the same
        }
    }
    float cx = -INFINITY;  // what is still possible: ranked before (cx, ci); at first all
    int ci = -1;
    for (;;) {
        double best = -1.0;
        int bi = none;
        for (int j = lane; j < V; j += NT) {
            const float v = s.x[j];
            if (s.r[j] > best && (v > cx || (v == cx && j < ci))) { best = s.r[j]; bi = j; }
        }
        J.best(best, bi);
        if (bi == none) return mi;  // (cannot be: the first of the order is always kept)
        const float vw = s.x[bi];
        int rank = 0;
        double S = 0.0;
        for (int j = lane; j < V; j += NT) {
            const float v = s.x[j];
            if (v > vw || (v == vw && j < bi)) { S += s.q[j]; ++rank; }
        }
        rank = J.isum(rank);
        if (rank == 0) return bi;
        S = J.sum(S);
        if (rank < rp.k && (!(rp.P < 1.f) || S < (double)rp.P * W) && !(s.q[bi] < (double)rp.m)) return bi;
        cx = vw;
        ci = bi;
    }
}
// Threads that read the row again in every pass, for any V.  Within the range of the 32-bit bounds the arg-max is looked for among
// the entries whose 32-bit ratio comes within twice the tolerance of the largest, usually one or two, and only those are
// evaluated in 64 bits.
template <typename T, int NT>
__device__ int64_t resolve_row64(const SampleArgs& a, int64_t row, int64_t b, uint32_t kth, double* sd, int* si) {
    Joint<NT> J{sd, si};
    const int lane = threadIdx.x & (NT - 1), V = a.V;
    const T* px = (const T*)a.x + row * a.ld;
    const float* u = a.u + row * a.ldu;
    auto score = [&](int j) { return to_f32<T>(px[j]); };
    const RowParams rp = row_params(a, b);
    const int none = INT32_MAX;
    // the first entry of the order
    double mxd = -1.0;  // (as an order key, so that one reduction serves)
    int mi = none;
#pragma unroll 4
    for (int j = lane; j < V; j += NT) {
        const uint32_t key = order_key(score(j));
        if (key && (double)key > mxd) { mxd = (double)key; mi = j; }
    }
    J.best(mxd, mi);
    if (mi == none) return row_empty(a);
    if (!(rp.T > 0.f)) return mi;  // greedy
    const uint32_t kmax = (uint32_t)mxd;
    const float mxf = score(mi) + 0.0f;
    const double mx = (double)mxf, rT = (double)rp.T;
    const bool top_inf = isinf(mx);
    auto weight = [&](uint32_t key, float v) -> double {
        if (key == kmax) return 1.0;
        return top_inf ? 0.0 : exp(((double)v - mx) / rT);
    };
    auto ratio = [&](uint32_t key, float v, int j) { return weight(key, v) / (1e-10 - log((double)noise_arg(u[j]))); };
    bool beyond = top_inf;
    const float c = rate_of(rp.T, beyond);
    const bool fast = !beyond;
    // mass of the k first of the order (when it is needed)
    double W = -1.0;
    auto mass = [&]() {
        uint32_t t = kth;
        if (!kth && rp.k < V) {  // the k-th largest key; 0 if there are no k candidates
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t ct = t | (1u << bit);
                int n = 0;
#pragma unroll 4
                for (int j = lane; j < V; j += NT) n += order_key(score(j)) >= ct;
                n = J.isum(n);
                if (n >= rp.k) t = ct;
                if (n == rp.k) break;  // (then exactly the k first are at or above t)
            }
        }
        double s = 0.0, q = 0.0;
        int n = 0;
#pragma unroll 4
        for (int j = lane; j < V; j += NT) {
            const float v = score(j);
            const uint32_t key = order_key(v);
            if (key > t) { s += weight(key, v); ++n; }
            else if (key == t && t) q = weight(key, v);
        }
        W = J.sum(s);
        if (t) {
            n = J.isum(n);
            int dummy = 0;
            J.best(q, dummy);
            W += (double)(rp.k - n) * q;  // of equal entries at the border the lowest indices are in; they weigh the same
        }
    };
    uint32_t kc = 0xffffffffu;  // what is still possible: ranked before (kc, ic)
    int ic = none;
    for (;;) {
        double bv = -1.0, least = -1.0;
        int bi = none;
        auto possible = [&](uint32_t key, int j) { return key && (key > kc || (key == kc && j < ic) || ic == none); };
        auto ratio32 = [&](float v, int j) { return (double)(__builtin_amdgcn_exp2f((v - mxf) * c) * inv_noise(u[j])); };
        if (fast) {
            int any = 0;
#pragma unroll 4
            for (int j = lane; j < V; j += NT) {
                const float v = score(j);
                const double r = ratio32(v, j);
                if (possible(order_key(v), j) && r > least) least = r;
            }
            J.best(least, any);
            least *= 1.0 - 2.0 * RATIO_TOL;
        }
#pragma unroll 4
        for (int j = lane; j < V; j += NT) {
            const float v = score(j);
            const uint32_t key = order_key(v);
            if (!possible(key, j) || (fast && ratio32(v, j) < least)) continue;
            const double r = ratio(key, v, j);
            if (r > bv) { bv = r; bi = j; }
        }
        J.best(bv, bi);
        if (bi == none) return mi;  // (cannot be: the first of the order is always kept)
        const float vw = score(bi);
        const uint32_t kw = order_key(vw);
        int rank = 0;
#pragma unroll 4
        for (int j = lane; j < V; j += NT) {
            const uint32_t key = order_key(score(j));
            rank += (key > kw) | ((key == kw) & (j < bi));
        }
        rank = J.isum(rank);
        if (rank == 0) return bi;
        if (rank < rp.k && !(weight(kw, vw) < (double)rp.m)) {
            if (!(rp.P < 1.f)) return bi;
            if (W < 0.0) mass();
            double S = 0.0;
#pragma unroll 4
            for (int j = lane; j < V; j += NT) {
                const float v = score(j);
                const uint32_t key = order_key(v);
                if (key > kw || (key == kw && j < bi)) S += weight(key, v);
            }
            if (J.sum(S) < (double)rp.P * W) return bi;
        }
        kc = kw;
        ic = bi;
    }
}

// ---- V <= 64: a lane owns a row.  Everything is register arithmetic over the lane's own entries, no cross-lane traffic; the
// rows of a wave are neighbours in memory, so the loads of a wave cover one stretch of it.  In the middle of a sampler run most
// rows are not sampled: a block packs those that are to its first lanes, and the waves behind them end.
// 524288 x 26 bf16: 21 us (86 MB, 4.1 TB/s), with top-p 34 us: there the compare and sum loops over the lane's entries bound it, of
// which all rows of a wave wait for the one with the most candidates to reject.  A wave per row took 5 times as long: 26 of 64
// lanes at work, and every sum and maximum six steps across lanes.
template <typename T, int VP> __device__ __forceinline__ void load_entries(const T* p, int V, float (&x)[VP]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < VP; c += E) {
        if (c + E <= VP && c + E <= V) {
            struct __attribute__((packed)) { T e[E]; } v;
            __builtin_memcpy(&v, p + c, 16);
#pragma unroll
            for (int i = 0; i < E; ++i) if (c + i < VP) x[c + i] = to_f32<T>(v.e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (c + i < VP) x[c + i] = c + i < V ? to_f32<T>(p[c + i]) : -INFINITY;
        }
    }
}

template <typename T, int VP>
__global__ void __launch_bounds__(256) sample_lane_kernel(SampleArgs a) {
    __shared__ int s_cnt;
    __shared__ uint8_t s_list[256];
    const int64_t row0 = (int64_t)blockIdx.x * 256;
    const bool per = a.T || a.P || a.m || a.k || a.move;
    const int64_t b0 = per ? (a.M < ((int64_t)1 << 31) ? (int64_t)((uint32_t)row0 / (uint32_t)(a.L < a.M ? a.L : a.M)) : row0 / a.L) : 0;
    const int64_t off0 = row0 - b0 * a.L;
    const int V = a.V, lane = threadIdx.x & 63;
    int r = threadIdx.x;
    bool on = row0 + r < a.M;
    auto batch_of = [&](int rr) -> int64_t {
        const int64_t q = off0 + rr;
        if (!per) return 0;
        return a.L >= 256 ? b0 + (q >= a.L) : b0 + (uint32_t)q / (uint32_t)a.L;
    };
    if (a.xcur) {  // (uniform: the barriers are met by the whole block)
        if (threadIdx.x == 0) s_cnt = 0;
        __syncthreads();
        bool go = false;
        if (on) {
            go = row_moves(a, row0 + r, a.move ? batch_of(r) : 0);
            if (!go) a.out[row0 + r] = a.xcur[row0 + r];
        }
        const unsigned long long mask = __ballot(go);
        int base = 0;
        if (lane == 0 && mask) base = atomicAdd(&s_cnt, __popcll(mask));
        base = __shfl(base, 0, 64);
        if (go) s_list[base + __popcll(mask & ((1ull << lane) - 1ull))] = (uint8_t)r;
        __syncthreads();
        on = (int)threadIdx.x < s_cnt;
        r = on ? s_list[threadIdx.x] : 0;
    }
    if (!__ballot(on)) return;
    const int64_t row = on ? row0 + r : row0, b = batch_of(on ? r : 0);
    const RowParams rp = row_params(a, b);
    float x[VP], ie[VP];
    load_entries<T, VP>((const T*)a.x + row * a.ld, V, x);
    load_entries<float, VP>(a.u + row * a.ldu, V, ie);
    float mx = -INFINITY;
    int mi = 0;
#pragma unroll
    for (int j = 0; j < VP; ++j) {
        x[j] = x[j] > -INFINITY ? x[j] : -INFINITY;  // (NaN is no candidate)
        mi = x[j] > mx ? j : mi;
        mx = fmaxf(mx, x[j]);
    }
    int got = -1;  // < 0: open;  the row's answer otherwise
    bool near = mx == INFINITY, open = on && mx > -INFINITY;
    const bool empty = !(mx > -INFINITY);
    if (!(rp.T > 0.f)) { got = mi; open = false; }
    const float c = rate_of(rp.T, near);
    near = near && open;
    open = open && !near;
    float b1 = -1.f, b2 = -1.f, xw = 0.f, W = 0.f;
    int iw = 0;
#pragma unroll
    for (int j = 0; j < VP; ++j) {
        const float q = __builtin_amdgcn_exp2f((x[j] - mx) * c);
        W += q;
        ie[j] = x[j] > -INFINITY ? q * inv_noise(ie[j]) : -1.f;  // the ratio takes the noise's place
        b2 = __builtin_amdgcn_fmed3f(b1, b2, ie[j]);
        iw = ie[j] > b1 ? j : iw;
        xw = ie[j] > b1 ? x[j] : xw;
        b1 = fmaxf(b1, ie[j]);
    }
    if (__ballot(open && rp.k < V && rp.P < 1.f)) {  // mass of the k first: the k-th largest value, bit by bit
        uint32_t t = 0;
        constexpr int LOW = sizeof(T) == 2 ? 16 : 0;
        bool exact = false;  // exactly k entries at or above t: lower bits change nothing
        for (int bit = 31; bit >= LOW; --bit) {
            const uint32_t ct = t | (1u << bit);
            const float tv = key_value(ct);
            int n = 0;
#pragma unroll
            for (int j = 0; j < VP; ++j) n += x[j] >= tv;
            if (!exact && n >= rp.k) { t = ct; exact = n == rp.k; }
            if (!__ballot(open && !exact)) break;
        }
        t = whole_key<LOW>(t);
        const float tv = key_value(t);
        float s = 0.f;
        int n = 0;
#pragma unroll
        for (int j = 0; j < VP; ++j) {
            const float q = __builtin_amdgcn_exp2f((x[j] - mx) * c);
            s += ((x[j] > tv) | (exact & (x[j] == tv))) ? q : 0.f;
            n += x[j] > tv;
        }
        if (t && rp.k < V) W = exact ? s : s + (float)(rp.k - n) * __builtin_amdgcn_exp2f((tv - mx) * c);
    }
    if (open && rp.k >= V && !(rp.P < 1.f) && !(rp.m > 0.f)) {  // nothing is cut off
        if (b2 < b1 * (1.f - RATIO_TOL)) got = iw;
        else near = true;
        open = false;
    }
    while (__ballot(open)) {
        float S = 0.f, n1 = -1.f, n2 = -1.f, nx = 0.f;
        int rank = 0, ni = 0;
#pragma unroll
        for (int j = 0; j < VP; ++j) {
            const bool before = (x[j] > xw) | ((x[j] == xw) & (j < iw));
            const float q = __builtin_amdgcn_exp2f((x[j] - mx) * c), v = before ? ie[j] : -1.f;
            S += before ? q : 0.f;
            rank += before;
            n2 = __builtin_amdgcn_fmed3f(n1, n2, v);
            ni = v > n1 ? j : ni;
            nx = v > n1 ? x[j] : nx;
            n1 = fmaxf(n1, v);
        }
        const Decision w = decide(rp, rank, S, W, __builtin_amdgcn_exp2f((xw - mx) * c), b1, b2);
        if (open && w != DROPPED) {
            open = false;
            if (w == KEPT) got = iw;
            else near = true;
        }
        b1 = n1; b2 = n2; iw = ni; xw = nx;
    }
    int64_t ans = empty ? row_empty(a) : (int64_t)got;
    for (unsigned long long todo = __ballot(near); todo; todo &= todo - 1) {
        const int src = __builtin_ctzll(todo);
        const int rr = __builtin_amdgcn_readlane(on ? r : 0, src);
        const int64_t v = resolve_lanes64<T>(a, row0 + rr, batch_of(rr));
        if (lane == src) ans = v;
    }
    if (on) a.out[row] = ans;
}

// ---- V > 64: NW waves own a row, its entries in registers (NE per lane, four neighbours at a time), so HBM is read once whatever
// the truncation.  16384 x 2365 bf16: 55 us (233 MB, 4.2 TB/s), top-k 50 59 us, top-p 0.9 82 us, both 66 us; the rest over the
// 46 us of the bytes is latency: a row's loads, its maximum, each rejection are one after the other, and 128 registers a lane leave
// four waves on a SIMD to cover them.
// the best and second best ratio, with the best one's value and index
struct Best {
    float b1, b2, x;
    int i;
};
// one lane's numbers joined over the NW waves of a row; every member is called by all of them.  The exchange alternates
// between two buffers, so a barrier per call is enough: a buffer is written again two calls later.
template <int NW> struct RowRed {
    float (*buf)[4 * NW];
    int turn = 0;
    __device__ __forceinline__ float max(float v) {
        v = dpp_max(v);
        if constexpr (NW > 1) {
            float* o = swap();
            if ((threadIdx.x & 63) == 0) o[threadIdx.x >> 6] = v;
            __syncthreads();
            v = dpp_max(o[threadIdx.x & (NW - 1)]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v) {
        v = dpp_sum(v);
        if constexpr (NW > 1) {
            float* o = swap();
            if ((threadIdx.x & 63) == 0) o[threadIdx.x >> 6] = v;
            __syncthreads();
            v = dpp_sum((threadIdx.x & 63) < NW ? o[threadIdx.x & (NW - 1)] : 0.f);
        }
        return v;
    }
    __device__ __forceinline__ int count(int n) {  // n is the wave's own (the same in all lanes)
        if constexpr (NW > 1) {
            float* o = swap();
            if ((threadIdx.x & 63) == 0) o[threadIdx.x >> 6] = (float)n;  // (below 2^24)
            __syncthreads();
            n = (int)dpp_sum((threadIdx.x & 63) < NW ? o[threadIdx.x & (NW - 1)] : 0.f);
        }
        return n;
    }
    // the best of all lanes
    __device__ __forceinline__ void best(Best& v) {
        pick(v, 64);
        if constexpr (NW > 1) {
            float* o = swap();
            const int w = threadIdx.x >> 6, l = threadIdx.x & (NW - 1);
            if ((threadIdx.x & 63) == 0) { o[w] = v.b1; o[NW + w] = v.b2; o[2 * NW + w] = v.x; o[3 * NW + w] = __int_as_float(v.i); }
            __syncthreads();
            v = {o[l], o[NW + l], o[2 * NW + l], __float_as_int(o[3 * NW + l])};
            pick(v, NW);
        }
    }
    // a sum over lanes and two counts of the wave
    __device__ __forceinline__ void sums(float& s, int& n, int& m) {
        s = dpp_sum(s);
        if constexpr (NW > 1) {
            float* o = swap();
            const int w = threadIdx.x >> 6, l = threadIdx.x & (NW - 1);
            if ((threadIdx.x & 63) == 0) { o[w] = s; o[NW + w] = (float)n; o[2 * NW + w] = (float)m; }
            __syncthreads();
            const bool mine = (threadIdx.x & 63) < NW;
            s = dpp_sum(mine ? o[l] : 0.f);
            n = (int)dpp_sum(mine ? o[NW + l] : 0.f);
            m = (int)dpp_sum(mine ? o[2 * NW + l] : 0.f);
        }
    }

  private:
    __device__ __forceinline__ float* swap() { turn ^= 1; return buf[turn]; }
    // the best of `n` different lanes (the wave holds them 64 / n times over).  Of equals any will do: the row is then near
    __device__ __forceinline__ void pick(Best& v, int n) {
        const float top = dpp_max(v.b1);
        const int src = __builtin_ctzll(__ballot(v.b1 == top));
        const bool won = ((int)(threadIdx.x & 63) & (n - 1)) == (src & (n - 1));
        const float second = dpp_max(won ? v.b2 : v.b1);
        v.x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v.x), src));
        v.i = __builtin_amdgcn_readlane(v.i, src);
        v.b1 = top;
        v.b2 = second;
    }
};
// the largest key t with at least k entries at or above it (0: there are not so many), bit by bit down to LOW; exactly k
// entries above a key end the search early.  Counts are popcounts of compare masks: no arithmetic across lanes.  With bits below
// LOW that are not known t is a bound: at least k entries reach it.
template <int LOW, int N, class R> __device__ __forceinline__ uint32_t kth_bits(const float (&x)[N], int k, R& red) {
    uint32_t t = 0;
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t ct = t | (1u << bit);
        const float tv = key_value(ct);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popcll(__ballot(x[i] >= tv));
        n = red.count(n);
        if (n >= k) {
            t = ct;
            if (n == k) break;
        }
    }
    return t;
}
// LOW 0, or 16 where the entries are bf16 numbers: the k-th key itself
template <int LOW, int N, class R> __device__ __forceinline__ uint32_t kth_key(const float (&x)[N], int k, R& red) {
    return whole_key<LOW>(kth_bits<LOW>(x, k, red));
}
// mass of the k first, where t is their kth_key
template <int N, class R>
__device__ __forceinline__ float mass_of_first(const float (&x)[N], int k, uint32_t t, float mx, float c, R& red) {
    const float tv = key_value(t);
    float s = 0.f, mm = mx;
    int n = 0;
    asm volatile("" : "+v"(mm));  // (not kept from the first pass, as in eliminate)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s += x[i] > tv ? __builtin_amdgcn_exp2f((x[i] - mm) * c) : 0.f;
        n += __popcll(__ballot(x[i] > tv));
    }
    s = red.sum(s);
    n = red.count(n);
    // the rest of the k lie at tv, or — where the search ended early — between tv and the next entry above it
    float at = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) at = fmaxf(at, x[i] == tv ? x[i] : -INFINITY);
    at = red.max(at);
    return at > -INFINITY ? s + (float)(k - n) * __builtin_amdgcn_exp2f((tv - mx) * c) : s;
}
// the best of the entries before (xw, index off + jw) — of all, if there is no such entry yet (xw = +inf)
template <int N, class R, class J>
__device__ __forceinline__ Best best_before(const float (&x)[N], const float (&r)[N], J jc, int off, float xw, int jw, bool tied, R& red) {
    Best v{-1.f, -1.f, 0.f, 0};
    if (tied) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float ri = (x[i] > xw) | ((x[i] == xw) & (jc(i) < jw)) ? r[i] : -1.f;
            v.b2 = __builtin_amdgcn_fmed3f(v.b1, v.b2, ri);
            v.i = ri > v.b1 ? i : v.i;
            v.x = ri > v.b1 ? x[i] : v.x;
            v.b1 = fmaxf(v.b1, ri);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float ri = x[i] > xw ? r[i] : -1.f;
            v.b2 = __builtin_amdgcn_fmed3f(v.b1, v.b2, ri);
            v.i = ri > v.b1 ? i : v.i;
            v.x = ri > v.b1 ? x[i] : v.x;
            v.b1 = fmaxf(v.b1, ri);
        }
    }
    v.i = off + jc(v.i);
    red.best(v);
    return v;
}
// the elimination over entries (x[i], index off + jc(i)) with ratios r[i] (-1: no candidate).  What a pass can compute again
// (the weights, the indexes) it does: kept from pass to pass it would take as many registers as the row.  Equal scores are
// rare, so the order among them costs a pass of its own when the candidate is not alone at its score.
template <bool RANK, int N, class R, class J>
__device__ __forceinline__ int eliminate(const RowParams& rp, bool cut, const float (&x)[N], const float (&r)[N], J jc, int off,
                                         float mx, float c, float W, R& red, bool& near) {
    Best v = best_before(x, r, jc, off, -INFINITY, 0, false, red);
    if (!cut) {
        near = !(v.b2 < v.b1 * (1.f - RATIO_TOL));
        return v.i;
    }
    for (;;) {
        float cc = c, mm = mx, s = 0.f;
        asm volatile("" : "+v"(cc), "+v"(mm));
        int above = 0, equal = 0, ties = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool gt = x[i] > v.x;
            s += gt ? __builtin_amdgcn_exp2f((x[i] - mm) * cc) : 0.f;
            if constexpr (RANK) above += __popcll(__ballot(gt));
            equal += __popcll(__ballot(x[i] == v.x));
        }
        red.sums(s, above, equal);
        const float q = __builtin_amdgcn_exp2f((v.x - mm) * cc);
        if (equal > 1) {
            const int vi = v.i - off;
#pragma unroll
            for (int i = 0; i < N; ++i) ties += __popcll(__ballot((x[i] == v.x) & (jc(i) < vi)));
            ties = red.count(ties);
            s += (float)ties * q;
        }
        const int rank = RANK ? above + ties : (v.x == mx ? ties : ties + 1);  // (without RANK only whether it is 0 matters)
        const Decision d = decide(rp, rank, s, W, q, v.b1, v.b2);
        if (d != DROPPED) {
            near = d == NEAR;
            return v.i;
        }
        v = best_before(x, r, jc, off, v.x, v.i - off, equal > 1, red);
    }
}

// Where top-k or min-p leaves few entries, they are packed, four to a lane of one wave, and only their noise is read:
// the k-th largest of the lanes' own maxima is a bound that at least k entries reach (k distinct lanes), usually not many more;
// its upper 16 bits do (488 x 32003 fp32, top-k 50: 42 us instead of 44; 14 bits pack too many at top-k 200: 81 us instead of 44).
#define PACK 256
template <int NW> struct WideShared {
    static constexpr int ROWS = NW == 1 ? 4 : 1;
    float x[ROWS][PACK];
    int j[ROWS][PACK];
    float red[2][4 * NW];
    int n, ans;
};
// the token of a row that is sampled; near: it is not settled; t: a key that separates the row's k first from the rest (the
// k-th largest, or one below it that exactly k entries of the row reach) if it was needed, else 0 (wave 0's is meant)
template <typename T, int NW, int NE>
__device__ __forceinline__ int64_t wide_row(const SampleArgs& a, int64_t row, int64_t b, WideShared<NW>& sh, bool& near, uint32_t& t) {
    constexpr int NT = NW * 64, LOW = sizeof(T) == 2 ? 16 : 0;
    const int V = a.V, lane = threadIdx.x & 63, tid = NW == 1 ? lane : (int)threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), slot = NW == 1 ? wave : 0;
    RowRed<NW> red{sh.red};
    RowRed<1> alone{nullptr};
    auto jof = [&](int i) { return (i >> 2) * (4 * NT) + tid * 4 + (i & 3); };
    {
        RowParams rp = row_params(a, b);
        const T* px = (const T*)a.x + row * a.ld;
        const float* pu = a.u + row * a.ldu;
        float x[NE], r[NE], top = -INFINITY;
        // the noise: at once where no truncation can pack the row, else when it is known what of it is read
        auto read_noise = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NE; i += 4) {
                const int j = jof(i);
                if (j + 4 <= V) {
                    struct __attribute__((packed)) { float e[4]; } v;
                    __builtin_memcpy(&v, pu + j, 16);
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[i + k] = v.e[k];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[i + k] = j + k < V ? pu[j + k] : 0.5f;
                }
            }
        };
        const bool whole = rp.k >= V && (rp.P < 1.f || !(rp.m > 0.f)) && rp.T > 0.f;
#pragma unroll
        for (int i = 0; i < NE; i += 4) {
            const int j = jof(i);
            if (j + 4 <= V) {
                struct __attribute__((packed)) { T e[4]; } v;
                __builtin_memcpy(&v, px + j, 4 * sizeof(T));
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i + k] = to_f32<T>(v.e[k]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i + k] = j + k < V ? to_f32<T>(px[j + k]) : -INFINITY;
            }
        }
        if (whole) read_noise();
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            x[i] = x[i] > -INFINITY ? x[i] : -INFINITY;
            top = fmaxf(top, x[i]);
        }
        const float mx = red.max(top);
        if (!(mx > -INFINITY)) return row_empty(a);
        near = mx == INFINITY;
        int got = -1;
        if (!(rp.T > 0.f)) {
            float first = -INFINITY;  // (an index is below 2^24)
#pragma unroll
            for (int i = NE - 1; i >= 0; --i) first = x[i] == mx ? -(float)jof(i) : first;
            got = (int)-red.max(first);
            near = false;
        } else {
            const float c = rate_of(rp.T, near);
            if (!near) {
                // a bound that what is kept reaches
                float thr = -INFINITY;
                int n = PACK + 1;
                uint32_t bound = 0;
                auto reach = [&]() __attribute__((always_inline)) {
                    int m = 0;
#pragma unroll
                    for (int i = 0; i < NE; ++i) m += __popcll(__ballot((x[i] >= thr) & (x[i] > -INFINITY)));
                    return m;
                };
                if (rp.k < V) {
                    if (rp.k <= PACK && rp.k <= NT) {
                        const float lm[1] = {top};
                        bound = kth_bits<16>(lm, rp.k, red);
                        if (bound) {
                            thr = key_value(bound);
                            n = red.count(reach());
                        }
                    }
                    if (n > PACK) {
                        t = kth_key<LOW>(x, rp.k, red);
                        if (t) thr = key_value(t);
                        else rp.k = V;  // (fewer candidates than k)
                        n = red.count(reach());
                    }
                } else if (!(rp.P < 1.f) && rp.m > 0.f) {
                    thr = fminf(mx + (__builtin_amdgcn_logf(rp.m) - 0.01f) / c, mx);  // (a min-p above 1 leaves the maximum)
                    n = red.count(reach());
                }
                const bool cut = rp.k < V || rp.P < 1.f || rp.m > 0.f;
                if (n <= PACK && (rp.k < V || !(rp.P < 1.f))) {
                    int base = 0;
                    if constexpr (NW > 1) {
                        if (threadIdx.x == 0) sh.n = 0;
                        __syncthreads();
                        const int mine = reach();
                        if (lane == 0) base = atomicAdd(&sh.n, mine);  // (the order of the packed entries does not matter)
                        base = __builtin_amdgcn_readfirstlane(base);
                    }
#pragma unroll
                    for (int i = 0; i < NE; ++i) {
                        const bool in = (x[i] >= thr) & (x[i] > -INFINITY);
                        const unsigned long long mask = __ballot(in);
                        if (in) {
                            const int at = base + __popcll(mask & ((1ull << lane) - 1ull));
                            sh.x[slot][at] = x[i];
                            sh.j[slot][at] = jof(i);
                        }
                        base += __popcll(mask);
                    }
                    if constexpr (NW > 1) __syncthreads();
                    else __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses are in order)
                    if (NW == 1 || wave == 0) {
                        float y[4], ry[4];
                        int jj[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int e = lane + 64 * i;
                            y[i] = e < n ? sh.x[slot][e] : -INFINITY;
                            jj[i] = e < n ? sh.j[slot][e] : 0;
                            ry[i] = e < n ? __builtin_amdgcn_exp2f((y[i] - mx) * c) * inv_noise(pu[jj[i]]) : -1.f;
                        }
                        float W = 0.f;
                        if (rp.P < 1.f) {
                            // Where exactly k entries are packed, the bound they reach is what separates them.  A search among
                            // them would end at the first key below them all, which more of the row may reach; of more than k
                            // it ends above the bound, where the packed entries are all that the row has.
                            if (!t) t = n == rp.k ? bound : kth_key<LOW>(y, rp.k, alone);
                            W = mass_of_first(y, rp.k, t, mx, c, alone);
                        }
                        got = eliminate<true, 4>(rp, cut, y, ry, [&](int i) { return i == 0 ? jj[0] : i == 1 ? jj[1] : i == 2 ? jj[2] : jj[3]; }, 0,
                                                 mx, c, W, alone, near);
                        if constexpr (NW > 1) {
                            if (lane == 0) sh.ans = near ? -1 : got;
                        }
                    }
                    if constexpr (NW > 1) {
                        __syncthreads();
                        got = sh.ans;
                        near = got < 0;
                    } else {
                        __builtin_amdgcn_wave_barrier();
                    }
                } else {
                    float W = 0.f;
                    if (!whole) read_noise();
#pragma unroll
                    for (int i = 0; i < NE; ++i) {
                        const float q = __builtin_amdgcn_exp2f((x[i] - mx) * c);
                        W += q;
                        r[i] = ((x[i] >= thr) & (x[i] > -INFINITY)) ? q * inv_noise(r[i]) : -1.f;
                    }
                    if (rp.P < 1.f) W = t ? mass_of_first(x, rp.k, t, mx, c, red) : red.sum(W);
                    auto jc = [&](int i) { return (i >> 2) * (4 * NT) + (i & 3); };
                    if (rp.k < V) got = eliminate<true, NE>(rp, cut, x, r, jc, tid * 4, mx, c, W, red, near);
                    else got = eliminate<false, NE>(rp, cut, x, r, jc, tid * 4, mx, c, W, red, near);
                }
            }
        }
        return got;
    }
}

// A row that came near gets this, and wide_row's t in the low half, in place of its token until sample_near_kernel, launched behind, has decided it: kept in this
// kernel, the 64-bit arithmetic would take its registers (115 instead of 60) and half of its waves (131072 x 300: 159 us with it,
// 79 us and 4 us for the launch behind without), and one wave alone with a row would be the last of the launch by 50 us.
#define NEAR_TOKEN INT64_MIN
template <typename T, int NW, int NE>
__global__ void __launch_bounds__(NW == 1 ? 256 : NW * 64, NE <= 40 ? 4 : 2) sample_wide_kernel(SampleArgs a) {
    __shared__ WideShared<NW> sh;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t row = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
    if (row >= a.M) return;
    const int64_t b = batch_of_row(a, row);
    bool near = false;
    uint32_t t = 0;
    const int64_t ans = row_moves(a, row, b) ? wide_row<T, NW, NE>(a, row, b, sh, near, t) : a.xcur[row];
    if (NW == 1 ? (threadIdx.x & 63) == 0 : threadIdx.x == 0) a.out[row] = near ? NEAR_TOKEN + (int64_t)t : ans;
}
// a block looks through `per` rows (at most 256) and takes those that came near one after the other
// 512 threads to a row: where a single row was sampled and its scores lie in the L2, a near row takes 6 us more than none at V = 2365
// and 11 us more at V = 9000 (256 threads: 8 and 20, 1024: 11 and 13).  Behind 16384 x 2365 bf16 the launch takes 4 to 5 us if no row
// is near, 12 to 16 with one (read from HBM) and 15 to 21 with three.
#define NEAR_NT 512
template <typename T, bool FITS> __global__ void __launch_bounds__(NEAR_NT) sample_near_kernel(SampleArgs a, int per) {
    constexpr int NT = NEAR_NT;
    __shared__ double sd[NT / 64];
    __shared__ int si[NT / 64];
    __shared__ uint64_t s_mask[NT / 64];
    __shared__ uint32_t s_kth[NT];
    const int64_t row0 = (int64_t)blockIdx.x * per, mine = row0 + threadIdx.x;
    const int64_t got = (int)threadIdx.x < per && mine < a.M ? a.out[mine] : 0;
    const bool near = got < NEAR_TOKEN + ((int64_t)1 << 32) && row_moves(a, mine, batch_of_row(a, mine));
    const uint64_t mask = __ballot(near);
    if ((threadIdx.x & 63) == 0) s_mask[threadIdx.x >> 6] = mask;
    s_kth[threadIdx.x] = (uint32_t)got;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        for (uint64_t todo = s_mask[w]; todo; todo &= todo - 1) {
            const int64_t row = row0 + w * 64 + __builtin_ctzll(todo), b = batch_of_row(a, row);
            const uint32_t kth = s_kth[row - row0];
            int64_t ans;
            if constexpr (FITS) {
                __shared__ StagedRow s_row;
                ans = resolve_staged64<T, NT>(a, row, b, kth, s_row, sd, si);
            } else {
                ans = resolve_row64<T, NT>(a, row, b, kth, sd, si);
            }
            if (threadIdx.x == 0) a.out[row] = ans;
        }
    }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_row64_kernel(SampleArgs a) {
    __shared__ double sd[NT / 64];
    __shared__ int si[NT / 64];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const int64_t b = batch_of_row(a, row);
        int64_t got;
        if (!row_moves(a, row, b)) got = a.xcur[row];
        else got = resolve_row64<T, NT>(a, row, b, 0, sd, si);
        if (threadIdx.x == 0) a.out[row] = got;
    }
}

template <typename T, int VP> static void launch_lane(const SampleArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((sample_lane_kernel<T, VP>), dim3((unsigned)((a.M + 255) / 256)), dim3(256), 0, st, a);
}
template <typename T, int NW, int NE> static void launch_wide(const SampleArgs& a, hipStream_t st) {
    constexpr int R = NW == 1 ? 4 : 1;
    hipLaunchKernelGGL((sample_wide_kernel<T, NW, NE>), dim3((unsigned)((a.M + R - 1) / R)), dim3(NW == 1 ? 256 : NW * 64), 0, st, a);
    int64_t per = (a.M + 255) / 256;  // (256 blocks; 512: a microsecond more where no row is near)
    per = per > 256 ? 256 : per;
    const dim3 grid((unsigned)((a.M + per - 1) / per));
    if (a.V <= STAGED) hipLaunchKernelGGL((sample_near_kernel<T, true>), grid, dim3(NEAR_NT), 0, st, a, (int)per);
    else hipLaunchKernelGGL((sample_near_kernel<T, false>), grid, dim3(NEAR_NT), 0, st, a, (int)per);
}
template <typename T> static void launch_sample(const SampleArgs& a, hipStream_t st) {
    // V up to a multiple of 4 (8 above 32): the entries behind V cost arithmetic, and a row is never read past its end
    if (a.V <= 4) launch_lane<T, 4>(a, st);
    else if (a.V <= 8) launch_lane<T, 8>(a, st);
    else if (a.V <= 12) launch_lane<T, 12>(a, st);
    else if (a.V <= 16) launch_lane<T, 16>(a, st);
    else if (a.V <= 20) launch_lane<T, 20>(a, st);
    else if (a.V <= 24) launch_lane<T, 24>(a, st);
    else if (a.V <= 28) launch_lane<T, 28>(a, st);
    else if (a.V <= 32) launch_lane<T, 32>(a, st);
    else if (a.V <= 40) launch_lane<T, 40>(a, st);
    else if (a.V <= 48) launch_lane<T, 48>(a, st);
    else if (a.V <= 64) launch_lane<T, 64>(a, st);
    // A wave per row up to 3000 entries, four waves up to 16384, sixteen up to 32768 (32 a lane: such a block has 128 registers
    // a lane).  Few rows leave most of the card idle and a pass over a row is what a call waits for: then four times the waves.
    // us, bf16, with top-p 0.3 | top-k 500 and top-p 0.3, one wave / four waves (V = 12000: four / sixteen):
    //   V =  2365:    64 rows 24 / 19 | 36 / 23;  512 rows 33 / 24 | 47 / 47;  2048 rows 46 / 43 | 59 / 85
    //   V =  3900:    64 rows 46 / 20 | 58 / 26;  512 rows 69 / 27 | 86 / 31;  8192 rows 188 / 105 | 248 / 196
    //   V = 12000:    64 rows 61 / 38 | 76 / 45;  256 rows 60 / 38 | 95 / 52;  2048 rows 218 / 174 | 274 / 405
    // (V = 600: no difference up to 512 rows.)
    // 40 entries a lane are the most for four waves on a SIMD (128 registers), 48 the most for three (167; 52 a lane leave two:
    // 392 us instead of 284 at V = 2900), and as far as that goes one wave is no worse where rows are many.  8192 rows, top-p 0.9 | top-p 0.3 |
    // top-k 500 and top-p 0.3 | top-k 50 and top-p 0.9, one wave / four waves:
    //   V = 1500:  39 / 41 |  79 / 77  |  79 / 102 | 31 / 63      V = 2365:  49 / 64 |  92 / 116 | 102 / 157 | 37 / 76
    //   V = 2560:  47 / 63 |  80 / 98  | 118 / 175 | 36 / 76      V = 2999:  77 / 80 | 124 / 124 | 137 / 158 | 66 / 93
    else if (a.V > 1024 && a.V <= 2048 && a.M <= 512) launch_wide<T, 4, 8>(a, st);
    else if (a.V > 2048 && a.V <= 4096 && (a.M <= 512 || a.V > 3000)) launch_wide<T, 4, 16>(a, st);
    else if (a.V > 4096 && a.V <= 8192 && a.M <= 256) launch_wide<T, 16, 8>(a, st);
    else if (a.V > 8192 && a.V <= 16384 && a.M <= 256) launch_wide<T, 16, 16>(a, st);
    else if (a.V <= 256) launch_wide<T, 1, 4>(a, st);
    else if (a.V <= 512) launch_wide<T, 1, 8>(a, st);
    else if (a.V <= 1024) launch_wide<T, 1, 16>(a, st);
    else if (a.V <= 2048) launch_wide<T, 1, 32>(a, st);
    else if (a.V <= 2560) launch_wide<T, 1, 40>(a, st);
    else if (a.V <= 3000) launch_wide<T, 1, 48>(a, st);
    else if (a.V <= 8192) launch_wide<T, 4, 32>(a, st);
    else if (a.V <= 16384) launch_wide<T, 4, 64>(a, st);
    else if (a.V <= 32768) launch_wide<T, 16, 32>(a, st);
    // A longer row does not fit a block's registers and is decided in 64 bits throughout, read again in every pass.  us, fp32, all
    // kept | top-p 0.9 | top-k 50 and top-p 0.9:  1 x 33001  37 | 62 | 156;  488 x 33001  122 | 325 | 680 (488 x 32003 above: 37 | 51 | 44);
    // 256 x 131071  237 | 726 | 1945
    else hipLaunchKernelGGL((sample_row64_kernel<T, 1024>), dim3(sedd_grid_for(a.M, 1, 512)), dim3(1024), 0, st, a);
}

extern "C" int sedd_sample_truncated(const void* logits, int dtype, int64_t ld, const float* u, int64_t ldu,
                                     const float* temperature, const int32_t* top_k, const float* top_p,
                                     const float* min_p, float temperature0, int top_k0, float top_p0, float min_p0,
                                     const int64_t* x, int64_t mask_id, const float* move, int64_t* out, int64_t M,
                                     int64_t L, int V, sedd_stream_t stream) {
    SEDD_CHECK_ARG(dtype == SEDD_F32 || dtype == SEDD_BF16, "sample_truncated: unknown dtype %d", dtype);
    SEDD_CHECK_ARG(M >= 0 && L > 0 && V > 0 && V <= 1 << 30 && M % L == 0, "sample_truncated: bad sizes M=%ld L=%ld V=%d", (long)M,
                   (long)L, V);
    // (a launch has at most 2^32 - 1 threads: 256 to four rows, or to one above 3000 entries, where memory ends before)
    SEDD_CHECK_ARG(M <= ((int64_t)1 << 26) - 4 || (V <= 64 && M <= ((int64_t)1 << 32) - 256), "sample_truncated: %ld rows of %d entries",
                   (long)M, V);
    SEDD_CHECK_ARG(M <= 1 || (ld >= V && ldu >= V + (move ? 1 : 0)), "sample_truncated: row strides %ld, %ld below V=%d",
                   (long)ld, (long)ldu, V);
    SEDD_CHECK_ARG(!move || x, "sample_truncated: move probabilities without current tokens");
    SEDD_CHECK_ARG(temperature || (temperature0 >= 0.f && temperature0 <= 3.402823466e38f),
                   "sample_truncated: temperature %f", (double)temperature0);
    SEDD_CHECK_ARG(top_p || (top_p0 >= 0.f && top_p0 <= 1.f), "sample_truncated: top_p %f not in [0, 1]", (double)top_p0);
    SEDD_CHECK_ARG(min_p || (min_p0 >= 0.f && min_p0 <= 1.f), "sample_truncated: min_p %f not in [0, 1]", (double)min_p0);
    SEDD_CHECK_ARG(top_k || top_k0 >= 0, "sample_truncated: top_k %d is negative", top_k0);
    if (M == 0) return SEDD_OK;
    SEDD_CHECK_ARG(logits && u && out, "sample_truncated: null pointer");
    SEDD_CHECK_ARG(out != x, "sample_truncated: out is x");  // (a row that came near is looked at again after out was written)
    const SampleArgs a{logits, ld, u, ldu, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0,
                       x, mask_id, move, out, M, L, V};
    if (dtype == SEDD_F32) launch_sample<float>(a, (hipStream_t)stream);
    else launch_sample<bf16_t>(a, (hipStream_t)stream);
    SEDD_LAUNCH_CHECK();
    return SEDD_OK;
}
