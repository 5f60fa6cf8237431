// fg_attention_kv8_tc.cu -- tree attention over the 8-bit KV cache on the
// tensor cores (bf16 models, head_dim 128).
//
// Both products run with the KV slots (or the head dims) as the 128 rows of
// the MMA and the query rows as its columns:
//   S^T [128 slots x R]  = K_tile [slots x dims] . Q^T       (K = 128 dims)
//   O^T [128 dims  x R] += V_tile^T [dims x slots] . P^T     (K = 128 slots)
// so an MMA's time follows the number of query rows R (32, 64, 96 or 128
// columns) instead of being that of 128 rows always, and the 32 lanes of a
// softmax warp are the 32 tokens of one 8-bit block: its two scales are
// warp-uniform scalars.
//
//   warps 0-3 / 4-7   softmax of the first / second half of the columns;
//                     thread = slot.  Row maxima are only ever needed when a
//                     weight exceeds the reference m of its column by more
//                     than 2^kGrow (the first tile, hardly ever later): a
//                     barrier with a vote decides, and only then are maxima
//                     taken across the slots, and O^T and l rescaled.  l
//                     stays per slot in registers until the end.
//   warps 8-11        V: e4m3 -> f16 (exact, by moving bits), from the staged
//                     codes into 128-byte-swizzled shared memory ([slot][dim]
//                     is the MN-major form that the transposed product reads)
//   warp 12           TMEM allocation; one thread issues tcgen05.mma
//   warp 13           TMA of the K and V codes, 16 KB a tile each
//
// K is multiplied as it is stored, in e4m3: Q enters as 2^a q = hi + lo, two
// e4m3 numbers of four bits each, 2^a the row's own (an element keeps its
// eight bits down to 2^-9 of the row's largest, behind that it is off by at
// most 2^-18 of it).  V and P are f16; what f16 lacks in range powers of two
// carry: P = 2^(x + lv - m + 3) for a score x (log2 domain) and a slot whose V
// has the scale 2^lv, m the column's largest x + lv up to 2^kGrow, so weights
// are kept relative to what they contribute to O, down to 2^-27 of it (a tail of 2^15 slots
// below that is at most 2^-12 of the result).  l =
// sum 2^(x - m) is fp32 and shares m; V's tiles hold value * 2^-8, so out =
// 32 O / l.  (Slots whose V scale is below 2^-100 contribute to l and not to
// O.)
//
// The tail's rows and the tree go through the same tiles: the slots of a row
// are numbered 0 .. q_len + tail_len + N - 1, tiles of 128 of them are read
// with the last, mixed, ones first.  A tail row gets a power of two of its own
// for K (hi + lo, like Q) and for V; slots past the end are zeros and masked.
// A query row with a NaN or an infinity has scores of NaN, and so has a tail
// slot whose K or V holds one, for the nodes that see it.
// Every mbarrier wait is bounded as in fg_attention_tc.cu; after a timeout a
// softmax warp runs on (so that the named barriers stay matched) and the CTA
// writes nothing.
//
// What bounds it: neither HBM nor the tensor pipe (8 MMAs take 380-530 clocks
// of a tile's ~2500) but the softmax warps' chain of TMEM load, vote,
// exponentials and stores per tile.  Measured at 64 query rows, 32 rows x 8
// heads x 16384 slots (1.09 GB, 168 us at the copy bandwidth): 354 us on keys
// with strong channels; the bf16 kernel on a bf16 cache of the same values
// (twice the bytes) 335 us.  The steps to it, on uniform codes, whose maxima
// hardly call for new references: K and V widened to bf16 from register
// prefetches 636 us (a release on a barrier waits for the loads a thread has in
// flight, so they hid nothing), TMA staging and scales in shared memory 360 us,
// plain try_wait 349 us, maxima by one redux each 344 us.  With more query rows
// per head the bf16 kernel is the faster one: 78 rows, 64 x 1024: 42.6 against
// 19.9 us; 224 rows, 16 x 2048: 65.4 against 30.8; with one node this one is:
// 254 against 329 us at 32 x 16384.
#include "fg_common.cuh"

namespace fg {
namespace kv8 {

using tc::bar_arrive;
using tc::bar_drain;
using tc::bar_init;
using tc::ex2;
using tc::fence_after;
using tc::fence_async_smem;
using tc::fence_before;
using tc::sa;
using tc::sdesc;
using tc::sw128;
using tc::umma;
using tc::umma_commit;

constexpr int kT = 128;                      // slots per tile
constexpr int kTcThreads = 512;             // 16 warps; of the last four two work
constexpr int kHalf = kT * 128;              // 16 KB: 128 rows of 128 bytes
constexpr int kTile = 2 * kHalf;             // an f16 V tile
constexpr int kMaxStages = 3;
constexpr int kScaleTiles = 256;  // tiles whose block scales a CTA keeps in shared memory
// Shared memory of the kernel for 32 NC columns: V tiles in f16 (32 KB each),
// two P buffers (f16, 64 columns per 16 KB), the rings of K and V codes (16 KB
// each), Q's two tiles, the block scales, the barriers and tables.
template <int NC>
struct Smem {
    static constexpr int kVBufs = NC <= 2 ? 2 : 1;
    static constexpr int kPBuf = NC <= 2 ? kHalf : kTile;
    static constexpr int kKStages = 3, kVStages = NC <= 2 ? 3 : 2;
    static constexpr int kOffV = 0, kOffP = kVBufs * kTile, kOffK = kOffP + 2 * kPBuf;
    static constexpr int kOffC = kOffK + kKStages * kHalf;  // V's codes
    static constexpr int kOffQ = kOffC + kVStages * kHalf, kOffScale = kOffQ + 2 * (32 * NC * 128);
    static constexpr int kOffBars = kOffScale + 2 * kScaleTiles * (kT / kBlk) * 4;
};
// P = 2^(d + lv + 3) with d + lv <= kGrow stays below 2^15; a smaller kGrow
// would keep weights further down and meet more maxima that call for new
// references (5 instead of 12 made the 64 x 1024 call half as slow again).
constexpr float kGrow = 12.0f;
constexpr float kNoMax = -1e30f;             // m of a column that has seen nothing

struct TcBars {
    uint64_t k_full[kMaxStages], k_empty[kMaxStages], c_full[kMaxStages], c_empty[kMaxStages];
    uint64_t v_full[2], v_empty[2];
    uint64_t s_full[2], p_full[2], p_free[2];
    uint64_t mix_full, mix_empty;  // K of a mixed tile
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
    float m_neg[128];    // minus the reference of each column, log2 domain
    float q_scale[128];  // the rows' 2^-a
    int32_t row_at[128];  // element offset of each query row behind the call row's first (of Q and out)
    float alpha[128];
    float wred[2][4][32];        // per half and warp: column maxima
    float tail_scale[2][4][kT];  // [K, V][step % 4]: the tail rows' scales
};
template <int NC>
constexpr int kTcSmem = Smem<NC>::kOffBars + (int)sizeof(TcBars) + 1024;
static_assert(kTcSmem<2> <= 232448 && kTcSmem<4> <= 232448, "shared memory of one CTA");

// f16 x f16 -> f32, M = 128; a_mn / b_mn: the operand's M / N index is the contiguous one
__host__ __device__ constexpr uint32_t idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kT >> 4) << 24);
}

// Codes are read once: they pass L1 by, which is what little the shared
// memory leaves of it.
__device__ __forceinline__ uint4 ldg_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// Bounded wait: false after about a second or when the CTA has aborted.  (One
// try per look at the clock: a waiting warp should take few issue slots.)
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag) {
    const uint32_t addr = sa(b);
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(addr), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        const uint64_t now = tc::gtime();
        if (t0 == 0) {
            t0 = now;
        } else if ((int64_t)(now - t0) > tc::kWaitNs) {
            *abort_flag = 1;
            atomicCAS(&g_fg_error_word, 0, FG_ETIMEOUT);
            return false;
        }
    }
}

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}

// Two fp32 operations per instruction, each rounded as the single one is.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r, x, y, z;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    memcpy(&z, &c, 8);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    memcpy(&a, &r, 8);
    return a;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r, x, y;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    memcpy(&a, &r, 8);
    return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r, x, y;
    memcpy(&x, &a, 8);
    memcpy(&y, &b, 8);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    memcpy(&a, &r, 8);
    return a;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Maximum over the warp's lanes (NaN is passed over) in one instruction.
__device__ __forceinline__ float lanes_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

template <int NREG>
__device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(NREG));
}
template <int NREG>
__device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(NREG));
}

template <int NC>
__device__ __forceinline__ void tld(uint32_t taddr, float* v);
template <>
__device__ __forceinline__ void tld<32>(uint32_t taddr, float* v) {
    tc::tld32(taddr, v);
}
template <>
__device__ __forceinline__ void tld<16>(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tst16(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
        "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
        "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])), "r"(__float_as_uint(v[8])),
        "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
        "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])),
        "r"(__float_as_uint(v[15]))
        : "memory");
}

// Four e4m3 codes to f16 pairs of value * 2^-8, elements (0, 2) and (1, 3):
// sign, exponent and mantissa are moved to where f16 has them, which leaves
// the exponent 8 short and maps subnormal codes to subnormal numbers.  (The
// conversion instruction becomes about five on this GPU; moving the bits
// takes 3.5 for two.)  A NaN code does not survive: its block's scale is NaN.
__device__ __forceinline__ void codes_to_f16_pairs(uint32_t w, uint32_t& even, uint32_t& odd) {
    even = ((w * 128u) & 0x3f803f80u) | ((w * 256u) & 0x80008000u);
    odd = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
}
// 16 codes; word k's elements land in the order 0, 2, 1, 3, which the output's
// dims undo at the end.
__device__ __forceinline__ void widen(const uint4& u, uint4& lo, uint4& hi) {
    codes_to_f16_pairs(u.x, lo.x, lo.y);
    codes_to_f16_pairs(u.y, lo.z, lo.w);
    codes_to_f16_pairs(u.z, hi.x, hi.y);
    codes_to_f16_pairs(u.w, hi.z, hi.w);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Elements (0, 2) and (1, 3) of four bf16 numbers times a power of two, as f16.
__device__ __forceinline__ uint32_t scale_even(uint32_t a, uint32_t b, float f) {
    return pack_f16(__uint_as_float(a << 16) * f, __uint_as_float(b << 16) * f);
}
__device__ __forceinline__ uint32_t scale_odd(uint32_t a, uint32_t b, float f) {
    return pack_f16(__uint_as_float(a & 0xffff0000u) * f, __uint_as_float(b & 0xffff0000u) * f);
}
// Four bf16 numbers times a power of two f as hi + lo in e4m3: eight bits are
// two times four, so the sum is exact for elements down to 2^-10 of the
// largest that fills the range, and off by at most 2^-10 behind that.
__device__ __forceinline__ void split_e4m3(uint2 w, float f, uint32_t& hi, uint32_t& lo) {
    const float x[4] = {__uint_as_float(w.x << 16) * f, __uint_as_float(w.x & 0xffff0000u) * f,
                        __uint_as_float(w.y << 16) * f, __uint_as_float(w.y & 0xffff0000u) * f};
    hi = lo = 0;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t h = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
        const __half2_raw back = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3);
        const float2 bf = __half22float2(__half2(back));
        const uint32_t l =
            __nv_cvt_float2_to_fp8x2(make_float2(x[i] - bf.x, x[i + 1] - bf.y), __NV_SATFINITE, __NV_E4M3);
        hi |= h << (8 * i);
        lo |= l << (8 * i);
    }
}
__device__ __forceinline__ uint32_t pair_mag(uint32_t w) {  // the larger magnitude of a bf16 pair, as fp32 bits
    return max((w << 16) & 0x7fffffffu, w & 0x7fff0000u);
}
// 2^e that brings a largest magnitude (fp32 bits) times 2^-e into [2^7, 2^8);
// 1 for zero, NaN for NaN and infinities (e4m3 and f16 would saturate those).
__device__ __forceinline__ float fp8_scale_of(uint32_t mag) {
    const int ex = (int)(mag >> 23);
    if (ex == 0) return 1.0f;
    if (ex == 255) return __int_as_float(0x7fffffff);
    return __uint_as_float((uint32_t)max(ex - 7, 1) << 23);
}

__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(
            tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* b) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(sa(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(sa(b))
        : "memory");
}

__device__ __forceinline__ bool group_any(int id, bool pred) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)pred), "r"(id)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// NC: 16-column chunks per half (R <= 32 NC query rows).
template <int NC>
__global__ void __launch_bounds__(kTcThreads, 1) attn_kv8_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                                    const __grid_constant__ CUtensorMap tm_v,
                                                                    const AttnParams p) {
    constexpr int H = 16 * NC, R2 = 2 * H;  // columns per half, of the MMA
    constexpr uint32_t kColO = 2 * R2;      // TMEM: S^T of even / odd tiles at 0 / R2, O^T
    constexpr uint32_t kCols = NC == 1 ? 128 : NC == 2 ? 256 : 512;
    static_assert(3 * R2 <= (int)kCols, "TMEM columns");
    // registers: 128 a thread at launch, 512 per lane slot of the four warps
    // of a scheduler; the softmax keeps H sums.  (A spilled register costs a trip to L2: the streams leave
    // nothing of the little L1.  The forms for more than 32 query rows spill 12 bytes and load 76 to 84.)
    constexpr int kRegSoft = 176, kRegConv = 96, kRegMma = 64;
    static_assert(2 * kRegSoft + kRegConv + kRegMma <= 512, "register split");
    constexpr int kKStages = Smem<NC>::kKStages, kOffVRing = Smem<NC>::kOffV, kOffPBuf = Smem<NC>::kOffP;
    constexpr int kOffKRing = Smem<NC>::kOffK, kOffQBuf = Smem<NC>::kOffQ, kPBuf = Smem<NC>::kPBuf;
    constexpr int kVBufs = Smem<NC>::kVBufs, kVStages = Smem<NC>::kVStages, kOffCodes = Smem<NC>::kOffC;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (sa(smem_raw) & 1023u)) & 1023u);  // (an offset: stays a shared address)
    TcBars* bars = reinterpret_cast<TcBars*>(smem + Smem<NC>::kOffBars);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, kvh = blockIdx.y / p.groups, grp = blockIdx.y % p.groups, b = blockIdx.z;
    const int row0 = grp * p.group_rows, R = min(p.group_rows, p.rows_total - row0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            bar_init(&bars->k_full[s], 1);
            bar_init(&bars->k_empty[s], 1);
            bar_init(&bars->c_full[s], 1);
            bar_init(&bars->c_empty[s], 4);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(&bars->v_full[s], 4);
            bar_init(&bars->v_empty[s], 1);
            bar_init(&bars->s_full[s], 1);
            bar_init(&bars->p_full[s], 8);
            bar_init(&bars->p_free[s], 1);
        }
        bar_init(&bars->mix_full, 4);
        bar_init(&bars->mix_empty, 1);
        bar_init(&bars->drain, 1);
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 128) {
        bars->m_neg[threadIdx.x] = -kNoMax;
        const int rr = row0 + min((int)threadIdx.x, R - 1);
        bars->row_at[threadIdx.x] = ((rr / p.G) * p.Hq + kvh * p.G + rr % p.G) * 128;
    }
    __syncthreads();
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sa(&bars->tmem_base)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // lengths, cache and Q may come from the preceding kernel
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const RowLens len = row_lens(p, b);
    const int64_t head = (int64_t)len.row * p.Hkv + kvh;
    const int T = len.q + len.t + p.N;
    const int nblk = (T + kT - 1) / kT;
    const int per = (nblk + p.splits - 1) / p.splits;
    const int c0 = min(nblk, split * per), c1 = min(nblk, c0 + per);
    const int nmine = c1 - c0;
    // tile of step i: from the last one down, so that the mixed tiles (from q_len on) come first
    const int nmixed = c1 - max(c0, min(c1, len.q / kT));
    auto tile_of = [&](int i) { return c1 - 1 - i; };

    // The first mixed tile's row of K and of V that this thread shares with
    // three others, and Q: all loads are in flight before any is used.
    // Pieces of a row: dims 64 s + 16 q + 8 x at u[2 s + x], or codes at u[0], u[2].
    auto load_mixed = [&](int i, int row, bool is_v, uint4* u) {
        const int slot = tile_of(i) * kT + row, q = lane & 3;
#pragma unroll
        for (int x = 0; x < 4; ++x) u[x] = make_uint4(0, 0, 0, 0);
        if (slot < len.q) {
            const uint8_t* src = (is_v ? p.v8 : p.k8) + (head * p.cap + slot) * 128 + q * 16;
            u[0] = ldg_stream(src);
            u[2] = ldg_stream(src + 64);
        } else if (slot < T) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(is_v ? p.vt : p.kt) +
                                                              (head * p.tcap + slot - len.q) * 128 + q * 16);
#pragma unroll
            for (int x = 0; x < 4; ++x) u[x] = src[(x >> 1) * 8 + (x & 1)];
        }
    };
    // ... to the tiles: V as code * 2^-8 in f16, K as hi + lo in e4m3; a tail row's scale to the table
    auto store_mixed = [&](int i, int row, bool is_v, const uint4* u) {
        const int q = lane & 3;
        const bool tail = tile_of(i) * kT + row >= len.q;
        uint32_t mag = 0;
        if (tail) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                mag = max(mag, max(max(pair_mag(u[x].x), pair_mag(u[x].y)), max(pair_mag(u[x].z), pair_mag(u[x].w))));
        }
        __syncwarp();
        mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
        mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
        const float sc = fp8_scale_of(mag), inv = inverse_pow2(sc);
        if (q == 0) bars->tail_scale[is_v][i & 3][row] = sc;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint4 a = u[2 * s], c = u[2 * s + 1];
            if (is_v) {
                uint4 lo, hi;
                if (tail && sc != sc) {
                    // zeros: the slot's score becomes NaN instead, which
                    // only the nodes that see it get
                    lo = hi = make_uint4(0, 0, 0, 0);
                } else if (tail) {
                    const float f = inv * 0x1p-8f;
                    lo = make_uint4(scale_even(a.x, a.y, f), scale_odd(a.x, a.y, f), scale_even(a.z, a.w, f),
                                    scale_odd(a.z, a.w, f));
                    hi = make_uint4(scale_even(c.x, c.y, f), scale_odd(c.x, c.y, f), scale_even(c.z, c.w, f),
                                    scale_odd(c.z, c.w, f));
                } else {
                    widen(a, lo, hi);
                }
                uint8_t* dst = smem + kOffVRing + (i % kVBufs) * kTile + s * kHalf;
                *reinterpret_cast<uint4*>(dst + sw128(row, 2 * q)) = lo;
                *reinterpret_cast<uint4*>(dst + sw128(row, 2 * q + 1)) = hi;
            } else {
                uint4 hi = a, lo = make_uint4(0, 0, 0, 0);
                if (tail) {
                    split_e4m3(make_uint2(a.x, a.y), inv, hi.x, lo.x);
                    split_e4m3(make_uint2(a.z, a.w), inv, hi.y, lo.y);
                    split_e4m3(make_uint2(c.x, c.y), inv, hi.z, lo.z);
                    split_e4m3(make_uint2(c.z, c.w), inv, hi.w, lo.w);
                }
                uint8_t* dst = smem + kOffKRing + sw128(row, 4 * s + q);
                *reinterpret_cast<uint4*>(dst) = hi;
                *reinterpret_cast<uint4*>(dst + kHalf) = lo;
            }
        }
    };
    {
        // Q's rows (zeros beyond R), kQ of them per warp: 2^a q = hi + lo in
        // e4m3, two tiles of 128-byte rows swizzled like the K tiles
        constexpr int kQ = R2 / (kTcThreads / 32);
        const __nv_bfloat16* q_base = static_cast<const __nv_bfloat16*>(p.q) + (int64_t)b * p.N * p.Hq * 128 + lane * 4;
        uint2 w[kQ];
#pragma unroll
        for (int x = 0; x < kQ; ++x) {
            const int r = warp * kQ + x;
            w[x] = make_uint2(0, 0);
            if (r < R) w[x] = *reinterpret_cast<const uint2*>(q_base + bars->row_at[r]);
        }
        // the block scales of this CTA's whole tiles: [K, V][step - nmixed][block of the tile]
        float* table = reinterpret_cast<float*>(smem + Smem<NC>::kOffScale);
        const int n_scale = min(nmine - nmixed, kScaleTiles) * (kT / kBlk);
        for (int e = threadIdx.x; e < 2 * n_scale; e += kTcThreads) {
            const bool is_v = e >= n_scale;
            const int x = is_v ? e - n_scale : e;
            table[(is_v ? kScaleTiles * (kT / kBlk) : 0) + x] =
                __ldg((is_v ? p.vs : p.ks) + head * (p.cap / kBlk) + tile_of(nmixed + x / 4) * (kT / kBlk) + x % 4);
        }
        const int row = warp * 8 + (lane >> 2);
        uint4 uk[4], uv[4];
        if (nmixed > 0) {
            load_mixed(0, row, false, uk);
            load_mixed(0, row, true, uv);
        }
#pragma unroll
        for (int x = 0; x < kQ; ++x) {
            const int r = warp * kQ + x;
            const float sc = fp8_scale_of(__reduce_max_sync(0xffffffffu, max(pair_mag(w[x].x), pair_mag(w[x].y))));
            uint32_t hi, lo;
            split_e4m3(w[x], inverse_pow2(sc), hi, lo);
            const uint32_t at = sw128(r, lane >> 2) + (lane & 3) * 4;
            *reinterpret_cast<uint32_t*>(smem + kOffQBuf + at) = hi;
            *reinterpret_cast<uint32_t*>(smem + kOffQBuf + R2 * 128 + at) = lo;
            if (lane == 0) bars->q_scale[r] = sc;
        }
        if (nmixed > 0) {
            store_mixed(0, row, false, uk);
            store_mixed(0, row, true, uv);
        }
    }
    fence_async_smem();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bars->tmem_base;

    if (warp >= 8 && warp < 12) {
        // ------------------------- converters: V's codes to f16 in shared memory; K and V of mixed tiles
        if constexpr (kRegConv > 128) reg_inc<kRegConv>();
        if constexpr (kRegConv < 128) reg_dec<kRegConv>();
        // this thread's rows of a tile: 32 w + lane / 4 + 8 h, 16-byte pieces q and q + 4 of each
        const int q = lane & 3, r_first = (warp - 8) * 32 + (lane >> 2);
        auto v_free = [&](int i) {
            const bool ok = i < kVBufs || bar_wait(&bars->v_empty[i % kVBufs], (i / kVBufs - 1) & 1, abort_flag);
            return (bool)__all_sync(0xffffffffu, ok);
        };
        auto publish_v = [&](int i) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->v_full[i % kVBufs]);
        };
        bool ok = true;
        if (nmixed > 0 && lane == 0) {  // the first mixed tile is there (all threads brought it)
            bar_arrive(&bars->mix_full);
            bar_arrive(&bars->v_full[0]);
        }
        for (int i = 1; i < nmixed && ok; ++i) {  // further ones: long tails and large trees
            // K first, as S^T(i) is issued before PV(i - 1), which frees V's buffer; K's two tiles are free once
            // the mixed tile before has been multiplied
            ok = __all_sync(0xffffffffu, bar_wait(&bars->mix_empty, (i - 1) & 1, abort_flag));
            if (!ok) break;
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
                uint4 u[4];
                load_mixed(i, r_first + 8 * h, false, u);
                store_mixed(i, r_first + 8 * h, false, u);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->mix_full);
            ok = v_free(i);
            if (!ok) break;
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
                uint4 u[4];
                load_mixed(i, r_first + 8 * h, true, u);
                store_mixed(i, r_first + 8 * h, true, u);
            }
            publish_v(i);
        }
        for (int i = nmixed; i < nmine && ok; ++i) {
            const int j = i - nmixed, st = j % kVStages;
            ok = v_free(i) &&
                 __all_sync(0xffffffffu, bar_wait(&bars->c_full[st], (j / kVStages) & 1, abort_flag));
            if (!ok) break;
            const uint8_t* src = smem + kOffCodes + st * kHalf;
            uint8_t* dst = smem + kOffVRing + (i % kVBufs) * kTile;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = r_first + 8 * (e >> 1);
                uint4 lo, hi;
                widen(*reinterpret_cast<const uint4*>(src + sw128(row, 4 * (e & 1) + q)), lo, hi);
                *reinterpret_cast<uint4*>(dst + (e & 1) * kHalf + sw128(row, 2 * q)) = lo;
                *reinterpret_cast<uint4*>(dst + (e & 1) * kHalf + sw128(row, 2 * q + 1)) = hi;
            }
            publish_v(i);
            if (lane == 0) bar_arrive(&bars->c_empty[st]);
        }
    } else if (warp >= 12) {
        reg_dec<kRegMma>();
        const int n8 = nmine - nmixed;  // whole 8-bit tiles: the j-th of them is step nmixed + j
        if (warp == 13) {
            // -------------------------------- codes by TMA: K by lane 0, V by lane 1
            // (Loads into registers would not do: a thread's release on a
            // barrier waits for the loads that it has in flight.)  K's stages
            // from 2 on in turn: the mixed tiles use 0 and 1 first.
            if (lane < 2) {
                const bool is_v = lane == 1;
                const int n_st = is_v ? kVStages : kKStages, first = is_v ? 0 : 2;
                uint64_t* full = is_v ? bars->c_full : bars->k_full;
                uint64_t* empty = is_v ? bars->c_empty : bars->k_empty;
                int issued = 0;
                for (int j = 0; j < n8; ++j) {
                    const int s = (j + first) % n_st;
                    // uses of this stage before: the tiles and, for K's 0 and 1, the mixed ones
                    const int before = j / n_st + (!is_v && s < 2 && nmixed > 0 ? 1 : 0);
                    if (before > 0 && !bar_wait(&empty[s], (before - 1) & 1, abort_flag)) break;
                    tc::bar_expect(&full[s], kHalf);
                    tma_2d(smem + (is_v ? kOffCodes : kOffKRing) + s * kHalf, is_v ? &tm_v : &tm_k, 0,
                           (int)(head * p.cap) + tile_of(nmixed + j) * kT, &full[s]);
                    issued = j + 1;
                }
                // the last loads have landed before this CTA's shared memory goes away
                for (int j = max(0, issued - n_st); j < issued; ++j)
                    bar_drain(&full[(j + first) % n_st], (j / n_st) & 1);
            }
            __syncwarp();
        }
        // ------------------------------------------------------ MMA issuer
        // The whole warp walks the tiles and one elected thread issues: values
        // that are uniform over the warp keep the descriptors in uniform
        // registers (under a one-lane branch an MMA took twice as long to issue).
        if (warp == 12) {
            constexpr uint32_t id_qk = idesc(R2, false, false);  // e4m3 has the type code of f16
            constexpr uint32_t id_pv = idesc(R2, true, true);
            const uint32_t base = sa(smem);
            const uint64_t q_desc = sdesc(base + kOffQBuf, 16, 1024);
            const uint64_t k_desc = sdesc(base + kOffKRing, 16, 1024);
            const uint64_t v_desc = sdesc(base + kOffVRing, kHalf, 1024);
            const uint64_t p_desc = sdesc(base + kOffPBuf, kHalf, 1024);
            const bool one = elect_one();
            auto wait = [&](uint64_t* bar, int phase) {
                const bool ok = __all_sync(0xffffffffu, bar_wait(bar, phase & 1, abort_flag));
                fence_after();
                return ok;
            };
            // S^T(i) = K(i) (Q_hi + Q_lo)^T once K(i) is there; S^T(i - 2) has been read: its P is
            auto issue_qk = [&](int i) {
                const uint32_t d = tmem + (uint32_t)((i & 1) * R2);
                const bool mixed = i < nmixed;
                const int j = i - nmixed, s = (j + 2) % kKStages;
                if (!(mixed ? wait(&bars->mix_full, i) : wait(&bars->k_full[s], j / kKStages)))
                    return false;
                if (one) {
                    if (mixed) {  // K_hi + K_lo
#pragma unroll 1
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                umma_fp8(d, k_desc + (uint64_t)((x >> 1) * (kHalf >> 4) + 2 * kk),
                                         q_desc + (uint64_t)((x & 1) * (R2 * 128 >> 4) + 2 * kk), id_qk,
                                         (x > 0 || kk > 0) ? 1u : 0u);
                        umma_commit(&bars->s_full[i & 1]);
                        umma_commit(&bars->mix_empty);
                        if (i == nmixed - 1) {
                            umma_commit(&bars->k_empty[0]);
                            umma_commit(&bars->k_empty[1]);
                        }
                    } else {
                        const uint64_t a = k_desc + (uint64_t)(s * (kHalf >> 4));
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            umma_fp8(d, a + 2 * (kk & 3), q_desc + (uint64_t)((kk >> 2) * (R2 * 128 >> 4) + 2 * (kk & 3)),
                                     id_qk, kk > 0 ? 1u : 0u);
                        umma_commit(&bars->s_full[i & 1]);
                        umma_commit(&bars->k_empty[s]);
                    }
                }
                __syncwarp();
                return true;
            };
            bool ok = true;
            for (int i = 0; i < min(2, nmine) && ok; ++i) ok = issue_qk(i);
            for (int i = 0; i < nmine && ok; ++i) {
                // O^T += V(i)^T P(i)^T
                ok = wait(&bars->p_full[i & 1], i >> 1) && wait(&bars->v_full[i % kVBufs], i / kVBufs);
                if (!ok) break;
                if (one) {
                    const uint64_t v_off = (uint64_t)((i % kVBufs) * (kTile >> 4)), p_off = (uint64_t)((i & 1) * (kPBuf >> 4));
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        umma(tmem + kColO, v_desc + v_off + kk * (2048 >> 4), p_desc + p_off + kk * (2048 >> 4), id_pv,
                             (i > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(&bars->p_free[i & 1]);
                    umma_commit(&bars->v_empty[i % kVBufs]);
                }
                __syncwarp();
                if (i + 2 < nmine) ok = issue_qk(i + 2);
            }
            // everything issued has completed before TMEM is read or freed
            if (one) {
                umma_commit(&bars->drain);
                bar_drain(&bars->drain, 0);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        // -------------------------------------------- softmax, one half of the columns
        reg_inc<kRegSoft>();
        constexpr int CW = NC % 2 == 0 ? 32 : 16;  // columns per vote
        const int hf = warp >> 2, w4 = warp & 3, bar_id = 1 + hf;
        const uint32_t lane_addr = (uint32_t)(w4 * 32) << 16;
        const int col0 = hf * H;
        const float sc = p.scale * 1.4426950408889634f;
        float* m_neg = bars->m_neg + col0;
        const float* q_sc = bars->q_scale + col0;
        float* alpha = bars->alpha + col0;
        float2 l[H / 2];
#pragma unroll
        for (int j = 0; j < H / 2; ++j) l[j] = make_float2(0.0f, 0.0f);
        bool ok = true;
        const float* ksp = p.ks + head * (p.cap / kBlk);
        const float* vsp = p.vs + head * (p.cap / kBlk);
        // This warp's block of a whole tile has its scales in the table (a tile
        // behind the table's end, or an 8-bit block of a mixed tile, in the cache).
        const int nb8 = len.q / kBlk;
        const float* table = reinterpret_cast<const float*>(smem + Smem<NC>::kOffScale) + w4;
        for (int i = 0; i < nmine; ++i) {
            float kt = 1.0f, vt = 1.0f;  // this slot's scales
            const int j8 = i - nmixed;
            if (j8 >= 0 && j8 < kScaleTiles) {
                kt = table[j8 * (kT / kBlk)];
                vt = table[(kScaleTiles + j8) * (kT / kBlk)];
            } else {
                const int blk = tile_of(i) * (kT / kBlk) + w4;
                if (blk < nb8) {
                    kt = __ldg(ksp + blk);
                    vt = __ldg(vsp + blk);
                }
            }
            const int slot = tile_of(i) * kT + w4 * 32 + lane;
            // columns that do not see this slot (tiles with tree slots only)
            uint64_t hide = 0;
            if (tile_of(i) * kT + kT > len.q + len.t) {
                if (slot >= T) {
                    hide = ~0ull;
                } else if (slot >= len.q + len.t) {
                    const int x = slot - len.q - len.t;
                    hide = ~0ull;
                    int j = 0;
                    for (int node = (row0 + col0) / p.G; node < p.N && j < H; ++node) {  // its G columns, from j on
                        const int end = min((node + 1) * p.G - row0 - col0, H);
                        if ((__ldg(p.anc + node * 4 + (x >> 5)) >> (x & 31)) & 1u)
                            hide &= ~(((end - j >= 64) ? ~0ull : ((1ull << (end - j)) - 1)) << j);
                        j = end;
                    }
                }
            }
            const bool masked = __any_sync(0xffffffffu, hide != 0);
            ok = bar_wait(&bars->s_full[i & 1], (i >> 1) & 1, abort_flag) && ok;
            __syncwarp();
            fence_after();
            if (i < nmixed) {
                // tail rows have scales of their own: K's came with K (S^T is there), V's come with V
                ok = bar_wait(&bars->v_full[i % kVBufs], (i / kVBufs) & 1, abort_flag) && ok;
                __syncwarp();
                if (slot >= len.q && slot < T) {
                    kt = bars->tail_scale[0][i & 3][w4 * 32 + lane];
                    vt = bars->tail_scale[1][i & 3][w4 * 32 + lane];
                    if (vt != vt) {  // V holds a NaN or an infinity
                        kt = vt;
                        vt = 1.0f;
                    }
                }
            }
            const float kc = kt * sc;
            const float2 kc2 = make_float2(kc, kc);
            // V's scale 2^lv: P = 2^(d + lv + 3) for d = x - m, and d + lv <= kGrow
            const int lv = max((int)(__float_as_uint(vt) >> 23) - 127, -100);
            const float limit = kGrow - (float)lv;
            const float vf = lv > -100 ? vt * 8.0f : 0.0f;
            const float2 vc2 = make_float2(vf, vf);
            const uint32_t s_addr = tmem + lane_addr + (uint32_t)((i & 1) * R2 + col0);
            uint8_t* pbuf = smem + kOffPBuf + (i & 1) * kPBuf;
            // PV(i - 2) has read this P buffer
            if (i >= 2) ok = bar_wait(&bars->p_free[i & 1], ((i >> 1) - 1) & 1, abort_flag) && ok;
            __syncwarp();
#pragma unroll
            for (int ch = 0; ch < H / CW; ++ch) {
                float d[CW];
                auto load = [&]() {
                    tld<CW>(s_addr + ch * CW, d);
#pragma unroll
                    for (int j = 0; j < CW; j += 4) {
                        const float4 m4 = *reinterpret_cast<const float4*>(m_neg + ch * CW + j);
                        const float4 q4 = *reinterpret_cast<const float4*>(q_sc + ch * CW + j);
                        const float2 a = fma2(make_float2(d[j], d[j + 1]), mul2(kc2, make_float2(q4.x, q4.y)),
                                              make_float2(m4.x, m4.y));
                        const float2 c = fma2(make_float2(d[j + 2], d[j + 3]), mul2(kc2, make_float2(q4.z, q4.w)),
                                              make_float2(m4.z, m4.w));
                        d[j] = a.x;
                        d[j + 1] = a.y;
                        d[j + 2] = c.x;
                        d[j + 3] = c.y;
                    }
                    if (masked) {
                        const uint32_t hb = (uint32_t)(hide >> (ch * CW));
#pragma unroll
                        for (int j = 0; j < CW; ++j) d[j] = ((hb >> j) & 1u) ? -INFINITY : d[j];
                    }
                };
                load();
                float mx = fmaxf(d[0], d[1]);
#pragma unroll
                for (int j = 2; j < CW; j += 2) mx = max3(mx, d[j], d[j + 1]);
                if (group_any(bar_id, mx > limit)) {
                    // new references: the maxima over the tile's slots
#pragma unroll 1
                    for (int cc = 0; cc < CW; cc += 16) {
                        float x[16];
                        tld<16>(s_addr + ch * CW + cc, x);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            x[j] = fmaf(x[j], kc * q_sc[ch * CW + cc + j], (float)lv);
                            if (masked && ((hide >> (ch * CW + cc + j)) & 1u)) x[j] = -INFINITY;
                            x[j] = lanes_max(x[j]);
                            if (lane == 0) bars->wred[hf][w4][cc + j] = x[j];
                        }
                    }
                    group_sync(bar_id);
                    const int tg = w4 * 32 + lane;
                    if (tg < CW) {
                        const float* wr = &bars->wred[hf][0][tg];
                        const float tm = fmaxf(fmaxf(wr[0], wr[32]), fmaxf(wr[64], wr[96]));
                        const float old = -m_neg[ch * CW + tg], now = fmaxf(old, tm);
                        alpha[ch * CW + tg] = ex2(old - now);
                        m_neg[ch * CW + tg] = -now;
                    }
                    group_sync(bar_id);
#pragma unroll
                    for (int j = 0; j < CW / 2; ++j)
                        l[ch * CW / 2 + j] =
                            mul2(l[ch * CW / 2 + j], make_float2(alpha[ch * CW + 2 * j], alpha[ch * CW + 2 * j + 1]));
                    if (i > 0) {
                        // O^T holds the tiles up to i - 1: rescale once PV(i - 1) has completed
                        ok = bar_wait(&bars->p_free[(i - 1) & 1], ((i - 1) >> 1) & 1, abort_flag) && ok;
                        __syncwarp();
                        fence_after();
#pragma unroll 1
                        for (int cc = 0; cc < CW; cc += 16) {
                            float o[16];
                            const uint32_t o_addr = tmem + lane_addr + kColO + col0 + ch * CW + cc;
                            tld<16>(o_addr, o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] *= alpha[ch * CW + cc + j];
                            tst16(o_addr, o);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    load();
                }
                const int row = w4 * 32 + lane;
#pragma unroll
                for (int j = 0; j < CW; j += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float2 e = make_float2(ex2(d[j + 2 * u]), ex2(d[j + 2 * u + 1]));
                        float2& lj = l[(ch * CW + j) / 2 + u];
                        lj = add2(lj, e);
                        const float2 pe = mul2(e, vc2);
                        w[u] = pack_f16(pe.x, pe.y);
                    }
                    // P^T: row = slot, columns in 16-byte pieces of 8
                    const int pc = (col0 + ch * CW + j) / 8;
                    *reinterpret_cast<uint4*>(pbuf + (pc >> 3) * kHalf + sw128(row, pc & 7)) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            fence_async_smem();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->p_full[i & 1]);  // S^T(i) has been read, too
        }
        // ---- the last PV, the columns' sums over the slots, then the output
        if (nmine > 0) {
            ok = bar_wait(&bars->p_free[(nmine - 1) & 1], ((nmine - 1) >> 1) & 1, abort_flag) && ok;
            __syncwarp();
        }
        fence_after();
        // (the P buffers are dead once the last PV has completed)
        float* sums = reinterpret_cast<float*>(smem + kOffPBuf) + hf * 4 * H;  // [warp][column]
#pragma unroll
        for (int ch = 0; ch < NC; ++ch) {
            // sums of 16 columns over the 32 lanes: halving exchanges leave one column with each pair of lanes
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = j & 1 ? l[ch * 8 + j / 2].y : l[ch * 8 + j / 2].x;
#pragma unroll
            for (int n = 8; n > 0; n >>= 1) {
                const bool up = lane & (2 * n);
#pragma unroll
                for (int j = 0; j < n; ++j) {
                    const float give = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
                    v[j] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * n);
                }
            }
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
            if ((lane & 1) == 0) sums[w4 * H + ch * 16 + (lane >> 1)] = v[0];
        }
        group_sync(bar_id);
        const bool good = __all_sync(0xffffffffu, ok && *abort_flag == 0);
        // this thread's dim: V's columns hold every four dims in the order 0, 2, 1, 3
        const int d0 = w4 * 32 + ((lane & ~3) | ((lane & 1) << 1) | ((lane >> 1) & 1));
        const int64_t item = ((int64_t)b * p.Hkv + kvh) * p.groups + grp;
        float* wo = p.splits > 1 ? p.ws_o + ((item * p.splits + split) * p.group_rows) * 128 : nullptr;
        float* wml = p.splits > 1 ? p.ws_ml + (item * p.splits + split) * 2 * p.group_rows : nullptr;
#pragma unroll
        for (int ch = 0; ch < NC; ++ch) {
            float o[16];
            if (nmine > 0) {
                tld<16>(tmem + lane_addr + kColO + col0 + ch * 16, o);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = 0.0f;
            }
            if (!good) continue;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int cc = ch * 16 + j, r = col0 + cc;
                if (r >= R) break;
                const float lt = (sums[cc] + sums[H + cc]) + (sums[2 * H + cc] + sums[3 * H + cc]);
                if (p.splits > 1) {
                    wo[(int64_t)r * 128 + d0] = o[j];
                    if (d0 == 0) {
                        wml[r] = -m_neg[cc] * 0.693147180559945309f;
                        wml[p.group_rows + r] = 0.03125f * lt;
                    }
                } else {
                    // no visible slot: 0; a NaN shows
                    const float inv = lt > 0.0f ? 32.0f / lt : (lt == 0.0f ? 0.0f : lt);
                    static_cast<__nv_bfloat16*>(p.out)[(int64_t)b * p.N * p.Hq * 128 + bars->row_at[r] + d0] =
                        __float2bfloat16(o[j] * inv);
                }
            }
        }
        fence_before();
    }
    __syncthreads();
    fence_after();
    if (warp == 12)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

}  // namespace kv8
}  // namespace fg
