// fg_logprobs.cu -- log probabilities of given tokens with entropy and best
// alternatives, and the gradient of both with respect to the logits.
//
// With x = logits / T, m = max x, S0 = sum e^(x - m), S1 = sum e^(x - m) (x - m):
//   lse = m + ln S0,  logp = x_t - lse,  H = ln S0 - S1 / S0
// in one pass over the row: every thread keeps (m, S0, S1) of its entries in
// 32 bits and moves them to a new maximum m' with d = m - m':
//   S1' = (S1 + S0 d) e^d,  S0' = S0 e^d.
// Everything runs in the log2 domain (z = x log2 e), so an exponential is one
// ex2 and the scale 1 / T is folded into the multiplier.
#include <cfloat>

#include "fg_common.cuh"
#include "fg_sampler.cuh"
#include "fg_vec.cuh"

namespace fg {
namespace lp {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.442695040888963407f;

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A step between two maxima in the log2 domain, floored where its exponential
// is 0 anyway: from a masked entry's lowest value it would overflow to -inf,
// and S0 d e^d to NaN.
__device__ __forceinline__ float step_of(float from, float to, float c) { return fmaxf((from - to) * c, -200.0f); }

// (m, S0, S1) of a set of entries; m is the raw maximum (before the scale),
// the sums are in the log2 domain.  No entries (or only -inf): m = -inf, 0, 0.
struct State {
    float m, s0, s1;
};

__device__ __forceinline__ State merge(const State& a, const State& b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s0 + b.s0, 0.0f};  // keeps a NaN sum
    const float da = step_of(a.m, m, c), db = step_of(b.m, m, c);  // a state without entries has S0 = 0
    const float fa = ex2f(da), fb = ex2f(db);
    State r;
    r.m = m;
    r.s0 = a.s0 * fa + b.s0 * fb;
    r.s1 = (a.s1 + a.s0 * da) * fa + (b.s1 + b.s0 * db) * fb;
    return r;
}

__device__ __forceinline__ State warp_merge(State s, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        State t;
        t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        t.s0 = __shfl_xor_sync(0xffffffffu, s.s0, o);
        t.s1 = __shfl_xor_sync(0xffffffffu, s.s1, o);
        s = merge(s, t, c);
    }
    return s;
}

// Adds NV loaded entries (their maximum vm is known): one comparison against
// the running maximum for all of them.
template <int NV>
__device__ __forceinline__ void add(State& s, const float (&x)[NV], float vm, float c) {
    if (vm > s.m) {
        const float d = step_of(s.m, vm, c), f = ex2f(d);
        s.s1 = (s.s1 + s.s0 * d) * f;
        s.s0 *= f;
        s.m = vm;
    }
    if (s.m == -INFINITY) {  // only masked entries so far
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (x[i] != x[i]) s.s0 = x[i];  // a NaN poisons the sum
        return;
    }
    // (x - m) c rather than x c - m c: exactly 0 at the maximum, and no
    // overflow among entries of the type's lowest value
    float a0 = 0.0f, a1 = 0.0f, b0 = 0.0f, b1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float z = (x[i] - s.m) * c;
        const float e = ex2f(z);
        const float zc = fmaxf(z, -200.0f);  // a masked entry (-inf) adds 0, not 0 * inf
        if (i & 1) {
            a1 += e;
            b1 = fmaf(e, zc, b1);
        } else {
            a0 += e;
            b0 = fmaf(e, zc, b0);
        }
    }
    s.s0 += a0 + a1;
    s.s1 += b0 + b1;
}

// Maximum of the entries of one 16-byte vector (NaN is passed over).
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& u) {
    float f[Vec<T>::N];
    unpack<T>(u, f);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < Vec<T>::N; ++i) m = fmaxf(m, f[i]);
    return m;
}
template <>
__device__ __forceinline__ float vec_max<__nv_bfloat16>(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    __nv_bfloat162 h[4];
    memcpy(h, w, 16);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// The part of a row that one CTA reads: rank r of CL takes the r-th share of
// the row's aligned 16-byte vectors; the entries before the first vector
// belong to rank 0, those behind the last one to the last rank.
template <typename T>
struct Slice {
    const T* row;
    int32_t head, v0, v1, tail0, tail1;  // [0, head) | vectors [v0, v1) | [tail0, tail1)

    __device__ __forceinline__ Slice(const T* r, int32_t vocab, int rank, int cl) : row(r) {
        constexpr int NV = Vec<T>::N;
        const int32_t skip = min(vocab, (int32_t)(((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / sizeof(T)));
        const int32_t nv = (vocab - skip) / NV;
        head = rank == 0 ? skip : 0;
        v0 = (int32_t)((int64_t)nv * rank / cl);
        v1 = (int32_t)((int64_t)nv * (rank + 1) / cl);
        tail0 = skip + nv * NV;
        tail1 = rank == cl - 1 ? vocab : tail0;
        row0 = skip;
    }
    int32_t row0;  // entry of vector 0
    __device__ __forceinline__ uint4 load(int32_t v) const { return ldg16(row + row0 + (int64_t)v * Vec<T>::N); }
    __device__ __forceinline__ int32_t index(int32_t v) const { return row0 + v * Vec<T>::N; }
    // odd entries: thread t's entry, -1 when it has none
    __device__ __forceinline__ int32_t odd(int t) const {
        return t < head ? t : (t - head < tail1 - tail0 ? tail0 + t - head : -1);
    }
};

struct FwdParams {
    const void* logits;
    int64_t row_stride;
    int32_t vocab, n;
    const int32_t* rows;
    int32_t n_rows;
    const int32_t* tokens;
    float c, inv_t;  // log2 e / T, 1 / T
    float *logp, *entropy, *lse;
    int32_t k;
    int32_t* top_idx;
    float* top_logp;
};

// The row of entry i, or nullptr for a padded entry (token < 0) and for a
// token or row outside its range (FG_EINVAL recorded).
template <typename T>
__device__ __forceinline__ const T* entry_row(const void* logits, int64_t row_stride, int32_t vocab,
                                              const int32_t* rows, int32_t n_rows, int32_t i, int32_t tok) {
    if (tok < 0) return nullptr;
    const int32_t r = rows != nullptr ? rows[i] : i;
    if (tok >= vocab || r < 0 || r >= n_rows) {
        if (threadIdx.x == 0) atomicCAS(&g_fg_error_word, 0, FG_EINVAL);
        return nullptr;
    }
    return static_cast<const T*>(logits) + (int64_t)r * row_stride;
}

constexpr int kCap = 512;  // candidates of the k best per CTA

// One row per cluster of CL CTAs of NT threads (CL = 1: one CTA).
//   pass 1  (m, S0, S1) of the row, and the maxima of 32 groups of threads.
//   k best  tau, the k-th largest group maximum of a CTA (the largest of the
//           cluster's), has k entries of the row at or above it, so the k best
//           are among the entries >= tau: pass 2 (the row comes from L2)
//           collects those, and one warp picks the k best of each CTA, then of
//           all.  More than kCap of them (flat rows): k rounds over the row,
//           round j taking the best entry behind round j - 1's.
// (value descending, index ascending) is a total order, so the result does
// not depend on the order in which the entries were collected.
template <typename T, int NT, int CL>
__global__ void __launch_bounds__(NT) logprobs_kernel(const FwdParams p) {
    constexpr int NW = NT / 32, NV = Vec<T>::N, U = 4;
    __shared__ State red[NW];
    __shared__ State all[CL];        // rank 0's copy holds every CTA's state
    __shared__ float gmax[32];       // maxima of 32 groups of NT / 32 threads
    __shared__ float tau_all[CL];
    __shared__ float cv[kCap];
    __shared__ int32_t ci[kCap];
    __shared__ int32_t cn;
    __shared__ int32_t cn_all[CL];
    __shared__ float kv[CL * FG_MAX_TOPK];
    __shared__ int32_t ki[CL * FG_MAX_TOPK];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = CL > 1 ? (int)cl_rank() : 0;
    const int32_t i = blockIdx.x / CL;
    const int32_t tok = p.tokens[i];
    const T* row = entry_row<T>(p.logits, p.row_stride, p.vocab, p.rows, p.n_rows, i, tok);
    if (row == nullptr) {  // the whole cluster leaves
        if (rank == 0) {
            if (tid == 0) {
                p.logp[i] = 0.0f;
                if (p.entropy) p.entropy[i] = 0.0f;
                if (p.lse) p.lse[i] = 0.0f;
            }
            if (tid < p.k) {
                p.top_idx[(int64_t)i * p.k + tid] = -1;
                p.top_logp[(int64_t)i * p.k + tid] = 0.0f;
            }
        }
        return;
    }
    // the cluster's CTAs have all started before any of them writes into another's shared memory
    if (CL > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const Slice<T> sl(row, p.vocab, rank, CL);
    State s = {-INFINITY, 0.0f, 0.0f};
    for (int32_t v = sl.v0 + tid; v < sl.v1; v += U * NT) {
        uint4 u[U];
#pragma unroll
        for (int a = 0; a < U; ++a)
            if (v + a * NT < sl.v1) u[a] = sl.load(v + a * NT);
#pragma unroll
        for (int a = 0; a < U; ++a) {
            if (v + a * NT >= sl.v1) break;
            float f[NV];
            unpack<T>(u[a], f);
            add<NV>(s, f, vec_max<T>(u[a]), p.c);
        }
    }
    const int32_t odd = sl.odd(tid);
    if (odd >= 0) {
        const float f[1] = {to_f<T>(row[odd])};
        add<1>(s, f, f[0], p.c);
    }
    {
        float g = s.m;  // this thread's maximum
#pragma unroll
        for (int o = NT / 64; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (tid % (NT / 32) == 0) gmax[tid / (NT / 32)] = g;
    }
    s = warp_merge(s, p.c);
    if (lane == 0) red[warp] = s;
    if (tid == 0) cn = 0;
    __syncthreads();
    if (CL > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
        State t = lane < NW ? red[lane] : State{-INFINITY, 0.0f, 0.0f};
        t = warp_merge(t, p.c);
        if (p.k > 0) {
            // tau: the k-th largest group maximum
            float a = gmax[lane], tau = -INFINITY;
            for (int j = 0; j < p.k; ++j) {
                tau = warp_max(a);
                const unsigned who = __ballot_sync(0xffffffffu, a == tau);
                if (lane == __ffs(who) - 1) a = -INFINITY;
            }
            if (lane < CL) {
                if (CL > 1)
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cl_addr(&tau_all[rank], lane)), "f"(tau)
                                 : "memory");
                else
                    tau_all[0] = tau;
            }
        }
        if (lane < CL) {
            if (CL > 1) {
                const uint32_t dst = cl_addr(&all[rank], lane);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(t.m) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(t.s0) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(t.s1) : "memory");
            } else {
                all[0] = t;
            }
        }
    }
    if (CL > 1) cl_sync(); else __syncthreads();
    s = all[0];
#pragma unroll
    for (int r = 1; r < CL; ++r) s = merge(s, all[r], p.c);
    const float ls = log2f(s.s0);
    auto logp_of = [&](float x) { return ((x - s.m) * p.c - ls) * kLn2; };
    if (rank == 0 && tid == 0) {
        p.logp[i] = logp_of(to_f<T>(row[tok]));
        if (p.entropy) p.entropy[i] = (ls - s.s1 / s.s0) * kLn2;
        if (p.lse) p.lse[i] = fmaf(s.m, p.inv_t, ls * kLn2);
    }
    if (p.k == 0) return;
    float tau = tau_all[0];
#pragma unroll
    for (int r = 1; r < CL; ++r) tau = fmaxf(tau, tau_all[r]);
    auto offer = [&](float x, int32_t at) {
        if (x >= tau) {
            const int32_t slot = atomicAdd(&cn, 1);
            if (slot < kCap) {
                cv[slot] = x;
                ci[slot] = at;
            }
        }
    };
    for (int32_t v = sl.v0 + tid; v < sl.v1; v += U * NT) {
        uint4 u[U];
#pragma unroll
        for (int a = 0; a < U; ++a)
            if (v + a * NT < sl.v1) u[a] = sl.load(v + a * NT);
#pragma unroll
        for (int a = 0; a < U; ++a) {
            if (v + a * NT >= sl.v1) break;
            if (!(vec_max<T>(u[a]) >= tau)) continue;
            float f[NV];
            unpack<T>(u[a], f);
#pragma unroll
            for (int e = 0; e < NV; ++e) offer(f[e], sl.index(v + a * NT) + e);
        }
    }
    if (odd >= 0) offer(to_f<T>(row[odd]), odd);
    __syncthreads();
    bool flat = cn > kCap;
    if (CL > 1) {
        if (tid < CL) {
            const int32_t mine_n = cn;
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cl_addr(&cn_all[rank], tid)), "r"(mine_n)
                         : "memory");
        }
        cl_sync();
        flat = false;
#pragma unroll
        for (int r = 0; r < CL; ++r) flat |= cn_all[r] > kCap;
    }
    // rank `to`'s list entry j of rank r's k best
    auto put = [&](int j, float v, int32_t id) {
        if (CL > 1) {
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cl_addr(&kv[rank * FG_MAX_TOPK + j], 0)), "f"(v)
                         : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cl_addr(&ki[rank * FG_MAX_TOPK + j], 0)), "r"(id)
                         : "memory");
        } else {
            kv[j] = v;
            ki[j] = id;
        }
    };
    // the best of the list (values v, indices id of n entries) behind (lv, li), by one warp
    auto next_best = [&](const float* v, const int32_t* id, int n, float lv, int32_t li, float& bv, int32_t& bi) {
        bv = -INFINITY;
        bi = 0x7fffffff;
        for (int q = lane; q < n; q += 32)
            if (better(lv, li, v[q], id[q]) && better(v[q], id[q], bv, bi)) {
                bv = v[q];
                bi = id[q];
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (better(ov, oi, bv, bi)) {
                bv = ov;
                bi = oi;
            }
        }
    };
    if (!flat) {
        if (warp == 0) {
            float lv = INFINITY, bv;
            int32_t li = -1, bi;
            for (int j = 0; j < p.k; ++j) {
                next_best(cv, ci, cn, lv, li, bv, bi);
                if (lane == 0) put(j, bv, bi);
                lv = bv;
                li = bi;
            }
        }
    } else {
        float lv = INFINITY;
        int32_t li = -1;
        for (int j = 0; j < p.k; ++j) {
            float bv = -INFINITY;
            int32_t bi = 0x7fffffff;
            auto see = [&](float x, int32_t at) {
                if (better(lv, li, x, at) && better(x, at, bv, bi)) {
                    bv = x;
                    bi = at;
                }
            };
            for (int32_t v = sl.v0 + tid; v < sl.v1; v += NT) {
                float f[NV];
                unpack<T>(sl.load(v), f);
#pragma unroll
                for (int e = 0; e < NV; ++e) see(f[e], sl.index(v) + e);
            }
            if (odd >= 0) see(to_f<T>(row[odd]), odd);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
                const int32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
                if (better(ov, oi, bv, bi)) {
                    bv = ov;
                    bi = oi;
                }
            }
            __syncthreads();
            if (lane == 0) {
                cv[warp] = bv;
                ci[warp] = bi;
            }
            __syncthreads();
            bv = cv[0];
            bi = ci[0];
            for (int w = 1; w < NW; ++w)
                if (better(cv[w], ci[w], bv, bi)) {
                    bv = cv[w];
                    bi = ci[w];
                }
            if (tid == 0) put(j, bv, bi);
            lv = bv;
            li = bi;
        }
    }
    if (CL > 1) cl_sync(); else __syncthreads();
    if (rank == 0 && warp == 0) {
        // every rank's k best, in lists of FG_MAX_TOPK: the unused ends are packed away first
        float lv = INFINITY, bv;
        int32_t li = -1, bi;
        for (int j = lane; j < CL * FG_MAX_TOPK; j += 32)
            if (j % FG_MAX_TOPK >= p.k) {
                kv[j] = -INFINITY;
                ki[j] = 0x7fffffff;
            }
        __syncwarp();
        for (int j = 0; j < p.k; ++j) {
            next_best(kv, ki, CL * FG_MAX_TOPK, lv, li, bv, bi);
            if (lane == 0) {
                const bool none = bi == 0x7fffffff;  // fewer than k entries that are not NaN
                p.top_idx[(int64_t)i * p.k + j] = none ? -1 : bi;
                p.top_logp[(int64_t)i * p.k + j] = none ? __int_as_float(0x7fffffff) : logp_of(bv);
            }
            lv = bv;
            li = bi;
        }
    }
}

struct BwdParams {
    const void* logits;
    int64_t row_stride;
    int32_t vocab, n;
    const int32_t* tokens;
    float c, inv_t;
    const float *lse, *entropy, *g, *h;
    void* out;
    int64_t out_stride;
};

// d logits_i = [ g (1[i = t] - p_i) - h p_i (ln p_i + H) ] / T
//            = g 1[i = t] / T + p_i (A z_i + B),   z_i = log2 p_i,
// A = -h ln 2 / T, B = -(g + h H) / T.  p_i = 0: the term is p ln p = 0 (z
// may be -inf).
template <bool ENT>
__device__ __forceinline__ float grad_of(float x, float c, float lse2, float a, float b) {
    const float z = fmaf(x, c, -lse2);
    const float e = ex2f(z);
    return ENT ? e * fmaf(a, fmaxf(z, -200.0f), b) : e * b;
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float* f);
template <>
__device__ __forceinline__ uint4 pack<float>(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <>
__device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack<__half>(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kBT = 256;  // threads of a backward CTA
// (4096 x 151936 bf16 with the entropy's gradient: 374 us, its read and write
// at the copy bandwidth.)

// One share of a row's vectors per CTA (blockIdx.y of gridDim.y), read and
// written once with 16-byte accesses where input and output start at the
// same place of a 16-byte line, else entry by entry.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kBT) logprobs_backward_kernel(const BwdParams p) {
    constexpr int NV = Vec<T>::N, U = 4;
    const int tid = threadIdx.x, rank = blockIdx.y, cl = gridDim.y;
    const int32_t i = blockIdx.x;
    const int32_t tok = p.tokens[i];
    const T* row = entry_row<T>(p.logits, p.row_stride, p.vocab, nullptr, p.n, i, tok);
    T* out = static_cast<T*>(p.out) + (int64_t)i * p.out_stride;
    const bool live = row != nullptr;
    if (!live) row = out;  // a padded row: zeros, cut as the output lies
    float lse2 = 0.0f, a = 0.0f, b = 0.0f, gt = 0.0f;
    if (live) {
        const float g = p.g[i], h = ENT ? p.h[i] : 0.0f;
        lse2 = fminf(fmaxf(p.lse[i] * kLog2e, -FLT_MAX), FLT_MAX);
        if (p.lse[i] != p.lse[i]) lse2 = p.lse[i];  // of a row with a NaN: shows
        a = -h * kLn2 * p.inv_t;
        b = -(ENT ? g + h * p.entropy[i] : g) * p.inv_t;
        gt = g * p.inv_t;
    }
    auto one = [&](int32_t j) {
        float d = live ? grad_of<ENT>(to_f<T>(row[j]), p.c, lse2, a, b) : 0.0f;
        if (j == tok) d += gt;
        out[j] = T(d);
    };
    if ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) {
        const int32_t lo = (int32_t)((int64_t)p.vocab * rank / cl), hi = (int32_t)((int64_t)p.vocab * (rank + 1) / cl);
        for (int32_t j = lo + tid; j < hi; j += kBT) one(j);
        return;
    }
    const Slice<T> sl(row, p.vocab, rank, cl);
    T* obase = out + sl.row0;
    for (int32_t v = sl.v0 + tid; v < sl.v1; v += U * kBT) {
        uint4 u[U];
        if (live) {
#pragma unroll
            for (int q = 0; q < U; ++q)
                if (v + q * kBT < sl.v1) u[q] = *reinterpret_cast<const uint4*>(row + sl.row0 + (int64_t)(v + q * kBT) * NV);
        }
#pragma unroll
        for (int q = 0; q < U; ++q) {
            const int32_t w = v + q * kBT;
            if (w >= sl.v1) break;
            float f[NV];
            if (live) {
                unpack<T>(u[q], f);
#pragma unroll
                for (int e = 0; e < NV; ++e) f[e] = grad_of<ENT>(f[e], p.c, lse2, a, b);
                const int32_t at = tok - sl.index(w);
                if ((uint32_t)at < (uint32_t)NV) {
#pragma unroll
                    for (int e = 0; e < NV; ++e)
                        if (e == at) f[e] += gt;
                }
            } else {
#pragma unroll
                for (int e = 0; e < NV; ++e) f[e] = 0.0f;
            }
            *reinterpret_cast<uint4*>(obase + (int64_t)w * NV) = pack<T>(f);
        }
    }
    const int32_t odd = sl.odd(tid);
    if (odd >= 0) one(odd);
}

// Rows up to kShort vectors take one 128-thread CTA each; longer ones 512
// threads, and a cluster of CTAs per row while all of them fit on the SMs at
// once: eight up to 18 rows, two up to 74, one from there on (151936 bf16
// logits with four alternatives, us at 8 / 2 / 1 CTAs a row: 8 rows 12.4 / 15.1
// / 20.0, 18 rows 14.4 / 15.1 / 20.6, 37 rows 22.4 / 15.1 / 20.6, 74 rows 32.8
// / 15.8 / 21.3, 192 rows 70.6 / 35.6 / 32.2).  Four are not used: 13.1 at 18
// and 30 rows, 16.0 at 37; two would still be faster at 110 rows, 21.0 against
// 24.0.  The largest batch, 4096 rows, streams at 0.88 of the copy bandwidth,
// 220 us.
constexpr int kShort = 1024;

// The kernels multiply by log2 e / T: a T so small that this is infinite makes
// NaN of the maximum's 0.
static bool good_temperature(float t) { return t > 0.0f && t < INFINITY && kLog2e / t < INFINITY; }

template <typename T, int NT, int CL>
static cudaError_t launch_fwd(const FwdParams& p, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.n * CL);
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CL;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CL > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, NT, CL>, p);
}

template <typename T>
static cudaError_t forward(const FwdParams& p, cudaStream_t st) {
    if (p.vocab <= kShort * Vec<T>::N) return launch_fwd<T, 128, 1>(p, st);
    if (p.n <= 148 / 8) return launch_fwd<T, 512, 8>(p, st);
    if (p.n <= 148 / 2) return launch_fwd<T, 512, 2>(p, st);
    return launch_fwd<T, 512, 1>(p, st);
}

template <typename T>
static void backward(const BwdParams& p, cudaStream_t st) {
    const int64_t nv = (p.vocab + Vec<T>::N - 1) / Vec<T>::N;
    // shares of at least one pass of the CTA's threads, about eight CTAs per SM in all
    int64_t cl = (nv + 4 * kBT - 1) / (4 * kBT);
    cl = min(cl, max((int64_t)1, (int64_t)(8 * 148) / p.n));
    const dim3 grid((unsigned)p.n, (unsigned)cl);
    if (p.h)
        logprobs_backward_kernel<T, true><<<grid, kBT, 0, st>>>(p);
    else
        logprobs_backward_kernel<T, false><<<grid, kBT, 0, st>>>(p);
}

}  // namespace lp
}  // namespace fg

using namespace fg;

extern "C" fg_status fg_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, int32_t vocab,
                                       int32_t n_rows, const int32_t* rows, const int32_t* tokens, int32_t n,
                                       float temperature, float* logp, float* entropy, float* lse, int32_t k,
                                       int32_t* top_idx, float* top_logp, void* stream) {
    if (n == 0) return FG_OK;
    if (!logits || !tokens || !logp || n < 0 || vocab <= 0 || n_rows <= 0 || (row_stride < vocab && n_rows > 1) ||
        (!rows && n_rows < n) || !lp::good_temperature(temperature) || k < 0)
        return FG_EINVAL;
    if (dtype != FG_DTYPE_F32 && dtype != FG_DTYPE_BF16 && dtype != FG_DTYPE_F16) return FG_EINVAL;
    if (k > FG_MAX_TOPK || k > vocab) return FG_ECAPACITY;
    if (k > 0 && (!top_idx || !top_logp)) return FG_EINVAL;
    lp::FwdParams p = {logits, row_stride, vocab, n, rows, n_rows, tokens, lp::kLog2e / temperature,
                       1.0f / temperature, logp, entropy, lse, k, top_idx, top_logp};
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = dtype == FG_DTYPE_BF16  ? lp::forward<__nv_bfloat16>(p, st)
                          : dtype == FG_DTYPE_F16 ? lp::forward<__half>(p, st)
                                                  : lp::forward<float>(p, st);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return FG_ECUDA;
    }
    return launch_status();
}

extern "C" fg_status fg_token_logprobs_backward(const void* logits, int32_t dtype, int64_t row_stride, int32_t vocab,
                                                const int32_t* tokens, int32_t n, float temperature, const float* lse,
                                                const float* entropy, const float* grad_logp,
                                                const float* grad_entropy, void* grad_logits, int64_t grad_stride,
                                                void* stream) {
    if (n == 0) return FG_OK;
    if (!logits || !tokens || !lse || !grad_logp || !grad_logits || n < 0 || vocab <= 0 ||
        (n > 1 && (row_stride < vocab || grad_stride < vocab)) || !lp::good_temperature(temperature) ||
        (grad_entropy && !entropy))
        return FG_EINVAL;
    if (dtype != FG_DTYPE_F32 && dtype != FG_DTYPE_BF16 && dtype != FG_DTYPE_F16) return FG_EINVAL;
    // in place means the same rows at the same places; any other overlap is a race
    const int64_t esz = dtype == FG_DTYPE_F32 ? 4 : 2;
    const char *lo = (const char*)logits, *go = (const char*)grad_logits;
    const char* lend = lo + ((int64_t)(n - 1) * row_stride + vocab) * esz;
    const char* gend = go + ((int64_t)(n - 1) * grad_stride + vocab) * esz;
    if (lo < gend && go < lend && !(lo == go && (n == 1 || grad_stride == row_stride))) return FG_EINVAL;
    lp::BwdParams p = {logits, row_stride, vocab, n, tokens, lp::kLog2e / temperature, 1.0f / temperature,
                       lse, entropy, grad_logp, grad_entropy, grad_logits, grad_stride};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == FG_DTYPE_BF16)
        lp::backward<__nv_bfloat16>(p, st);
    else if (dtype == FG_DTYPE_F16)
        lp::backward<__half>(p, st);
    else
        lp::backward<float>(p, st);
    return launch_status();
}
