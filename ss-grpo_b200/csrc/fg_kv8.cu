// fg_kv8.cu -- the 8-bit KV cache: bulk load after a prefill, commit at the
// end of a round.
//
// A block of FG_KV8_BLOCK tokens of one (layer, row, KV head) is stored as
// e4m3 codes and one scale s = 2^e per block, e the smallest integer >= -126
// with max |x| <= 448 * 2^e: codes = RNE_e4m3(x * 2^-e).  A power of two
// costs e4m3 no precision against max / 448 (its codes are floating-point
// numbers), the product x * 2^-e is exact, and code * s is exact in bf16, so
// the stored value does not depend on any order of roundings.  A block that
// holds a NaN or an infinity gets the scale NaN: whatever attends to it shows
// it.
#include <cuda_fp8.h>

#include "fg_common.cuh"

namespace fg {
namespace kv8 {

constexpr int kBlk = FG_KV8_BLOCK;
constexpr int kNT = 128;
constexpr int kMaxD = 128;

// 2^e of a block with this maximum (see above); NaN for a NaN or infinite one.
__device__ __forceinline__ float block_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int ex = (int)(b >> 23);  // amax >= 0
    if (ex == 255) return __int_as_float(0x7fffffff);
    // amax = 1.f * 2^(ex - 127), 448 = 1.75 * 2^8
    int e = ex - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, -126);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// 1 / s for a power of two s in [2^-126, 2^120], exactly.
__device__ __forceinline__ float inverse_pow2(float s) {
    const uint32_t b = __float_as_uint(s);
    if ((b >> 23) == 255) return s;
    return __uint_as_float((254u << 23) - b);
}

// 16 elements of a row; the source is read with 16-byte loads where its
// address and strides allow it.
template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, float* f);
template <>
__device__ __forceinline__ void load16<float>(const float* p, bool vec, float* f) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(p)[i];
            f[4 * i] = v.x;
            f[4 * i + 1] = v.y;
            f[4 * i + 2] = v.z;
            f[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = p[i];
    }
}
template <>
__device__ __forceinline__ void load16<__nv_bfloat16>(const __nv_bfloat16* p, bool vec, float* f) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[i];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
                f[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __bfloat162float(p[i]);
    }
}

// 16 elements to a 16-byte aligned tail row.
__device__ __forceinline__ void store16(float* p, const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // the values came from bf16: the truncation is exact
            w[j] = (__float_as_uint(f[8 * i + 2 * j]) >> 16) | (__float_as_uint(f[8 * i + 2 * j + 1]) & 0xffff0000u);
        }
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ uint4 codes16(const float* f, float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
            make_float2(f[4 * i] * inv, f[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
            make_float2(f[4 * i + 2] * inv, f[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
        w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// |x| as an ordered integer: the maximum over these is the block's maximum,
// and a NaN (largest pattern) survives it, which fmaxf would drop.
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float block_max(uint32_t m, uint32_t* red) {
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    uint32_t r = red[0];
#pragma unroll
    for (int w = 1; w < kNT / 32; ++w) r = max(r, red[w]);
    __syncthreads();
    return __uint_as_float(r);
}

template <typename T>
struct Buf {
    uint8_t* codes;  // of K or V
    float* scale;
    T* tail;
    int32_t batch, hkv, D, cap, tcap;

    __device__ __forceinline__ int64_t head(int32_t layer, int32_t row, int32_t h) const {
        return ((int64_t)layer * batch + row) * hkv + h;
    }
};

// A 32 x D block is dealt to the threads in pieces of 16 elements: piece
// e = tid + i * kNT is token e / (D / 16), dims 16 (e % (D / 16)).
constexpr int kPieces = kBlk * kMaxD / 16 / kNT;  // pieces per thread at D = 128

// ------------------------------------------------------------------- load
// One CTA per (32-token block, head x {K, V}, source row); the block is read
// once and written to every repeat.  The block behind the last whole one
// holds the row's remaining tokens, which go to the tail.
template <typename T>
__global__ void __launch_bounds__(kNT) load_kernel(Buf<T> bk, Buf<T> bv, int32_t layer, const T* __restrict__ k,
                                                   const T* __restrict__ v, int64_t sb, int64_t sh, int64_t ss,
                                                   bool vec, int32_t S, const int32_t* __restrict__ lengths,
                                                   int32_t repeats, const int32_t* rows, int32_t* __restrict__ q_len,
                                                   int32_t* __restrict__ tail_len) {
    __shared__ uint32_t red[kNT / 32];
    const int32_t blk = blockIdx.x, p = blockIdx.z;
    const int32_t h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const Buf<T>& b = is_v ? bv : bk;
    const T* src = (is_v ? v : k) + (int64_t)p * sb + (int64_t)h * sh;
    int32_t len = lengths[p];
    if (len < 0 || len > S) {  // nothing of such a row is loaded
        if (threadIdx.x == 0) atomicCAS(&g_fg_error_word, 0, FG_EINVAL);
        len = 0;
    }
    const int32_t whole = len / kBlk, rest = len % kBlk;
    if (blk == 0 && blockIdx.y == 0)
        for (int32_t r = threadIdx.x; r < repeats; r += kNT) {
            const bool there = cache_row(rows, b.batch, p * repeats + r) >= 0;
            q_len[p * repeats + r] = there ? whole * kBlk : 0;
            tail_len[p * repeats + r] = there ? rest : 0;
        }
    if (blk > whole || (blk == whole && rest == 0)) return;
    const int per = b.D / 16, n = (blk == whole ? rest : kBlk) * per;
    float f[kPieces][16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int e = threadIdx.x + i * kNT;
        if (e < n) {
            load16<T>(src + (int64_t)(blk * kBlk + e / per) * ss + (e % per) * 16, vec, f[i]);
#pragma unroll
            for (int j = 0; j < 16; ++j) m = max(m, mag(f[i][j]));
        }
    }
    const float scale = blk < whole ? block_scale(block_max(m, red)) : 1.0f;
    const float inv = inverse_pow2(scale);
    for (int32_t r = 0; r < repeats; ++r) {
        const int32_t row = cache_row(rows, b.batch, p * repeats + r);
        if (row < 0) continue;
        const int64_t head = b.head(layer, row, h);
        if (blk < whole) {
            uint8_t* dst = b.codes + (head * b.cap + blk * kBlk) * b.D;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int e = threadIdx.x + i * kNT;
                if (e < n) reinterpret_cast<uint4*>(dst)[e] = codes16(f[i], inv);
            }
            if (threadIdx.x == 0) b.scale[head * (b.cap / kBlk) + blk] = scale;
        } else {
            T* dst = b.tail + head * b.tcap * b.D;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int e = threadIdx.x + i * kNT;
                if (e < n) store16(dst + e * 16, f[i]);
            }
        }
    }
}

// ----------------------------------------------------------------- commit
// What a row's commit does, from its lengths and path; every CTA of the row
// and the kernel that writes the lengths come to the same answer.
struct Commit {
    bool ok;         // false: the row stays as it is (error recorded)
    int32_t row;     // cache row
    int32_t q, t, a; // lengths before the commit, accepted tokens
    int32_t blocks, rest;
};

__device__ __forceinline__ Commit commit_of(int32_t b, const int32_t* q_len, const int32_t* tail_len,
                                            const int32_t* acc_nodes, int32_t dcap, const int32_t* acc_len,
                                            const int32_t* rows, int32_t batch, int32_t cap, int32_t tcap) {
    Commit c;
    c.row = cache_row(rows, batch, b);
    c.q = q_len[b];
    c.t = tail_len[b];
    c.a = acc_len[b];
    c.ok = c.row >= 0 && c.q >= 0 && c.q % kBlk == 0 && c.q <= cap && c.t >= 0 && c.t <= tcap && c.a >= 0 && c.a <= dcap &&
           c.a <= tcap - c.t;
    int err = c.ok ? FG_OK : FG_EINVAL;
    c.blocks = c.rest = 0;
    if (c.ok) {
        int32_t last = -1;
        for (int32_t j = 0; j < c.a; ++j) {  // a path: increasing nodes inside the tail
            const int32_t x = acc_nodes[(int64_t)b * dcap + j];
            if (x <= last || x >= tcap - c.t) err = FG_EINVAL;
            last = x;
        }
        c.blocks = (c.t + c.a) / kBlk;
        c.rest = (c.t + c.a) % kBlk;
        if (err == FG_OK && c.blocks * kBlk > cap - c.q) err = FG_ECAPACITY;
        c.ok = err == FG_OK;
    }
    if (!c.ok && threadIdx.x == 0) atomicCAS(&g_fg_error_word, 0, err);
    return c;
}

// One CTA per (layer, head x {K, V}, row).  Compact slot s < t + a is tail
// slot s (s < t) or t + node of the path's token s - t.
template <typename T>
__global__ void __launch_bounds__(kNT) commit_kernel(Buf<T> bk, Buf<T> bv, const int32_t* __restrict__ acc_nodes,
                                                     int32_t dcap, const int32_t* __restrict__ acc_len,
                                                     const int32_t* rows, const int32_t* q_len,
                                                     const int32_t* tail_len, int32_t* q_out, int32_t* t_out) {
    __shared__ uint32_t red[kNT / 32];
    __shared__ int32_t path[FG_MAX_PATH];
    const int32_t h = blockIdx.x >> 1, layer = blockIdx.y, b = blockIdx.z;
    const Buf<T>& buf = (blockIdx.x & 1) ? bv : bk;
    const Commit c = commit_of(b, q_len, tail_len, acc_nodes, dcap, acc_len, rows, buf.batch, buf.cap, buf.tcap);
    if (q_out != nullptr && blockIdx.x == 0 && layer == 0 && threadIdx.x == 0) {
        q_out[b] = c.q + c.blocks * kBlk * (c.ok ? 1 : 0);
        t_out[b] = c.ok ? c.rest : c.t;
    }
    if (!c.ok || (c.a == 0 && c.blocks == 0)) return;
    if (threadIdx.x < c.a) path[threadIdx.x] = acc_nodes[(int64_t)b * dcap + threadIdx.x];
    __syncthreads();
    const int64_t head = buf.head(layer, c.row, h);
    T* tail = buf.tail + head * buf.tcap * buf.D;
    const int per = buf.D / 16;
    auto slot_of = [&](int32_t s) { return s < c.t ? s : c.t + path[s - c.t]; };
    float f[kPieces][16];
    for (int32_t blk = 0; blk < c.blocks; ++blk) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = threadIdx.x + i * kNT;
            if (e < kBlk * per) {
                load16<T>(tail + (int64_t)slot_of(blk * kBlk + e / per) * buf.D + (e % per) * 16, true, f[i]);
#pragma unroll
                for (int j = 0; j < 16; ++j) m = max(m, mag(f[i][j]));
            }
        }
        const float scale = block_scale(block_max(m, red));
        const float inv = inverse_pow2(scale);
        uint8_t* dst = buf.codes + (head * buf.cap + c.q + blk * kBlk) * buf.D;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int e = threadIdx.x + i * kNT;
            if (e < kBlk * per) reinterpret_cast<uint4*>(dst)[e] = codes16(f[i], inv);
        }
        if (threadIdx.x == 0) buf.scale[head * (buf.cap / kBlk) + c.q / kBlk + blk] = scale;
    }
    // what remains moves to the tail's start: all of it is read before any of it is written
    const int first = c.blocks == 0 ? c.t * per : 0, n = c.rest * per;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int e = threadIdx.x + i * kNT;
        if (e >= first && e < n)
            load16<T>(tail + (int64_t)slot_of(c.blocks * kBlk + e / per) * buf.D + (e % per) * 16, true, f[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int e = threadIdx.x + i * kNT;
        if (e >= first && e < n) store16(tail + (int64_t)e * 16, f[i]);
    }
}

// The new lengths, where they replace the old ones: after every CTA of
// commit_kernel has read those.
__global__ void commit_lengths_kernel(const int32_t* acc_nodes, int32_t dcap, const int32_t* acc_len,
                                      const int32_t* rows, int32_t batch, int32_t cap, int32_t tcap, int32_t B,
                                      int32_t* q_len, int32_t* tail_len) {
    const int32_t b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= B) return;
    const Commit c = commit_of(b, q_len, tail_len, acc_nodes, dcap, acc_len, rows, batch, cap, tcap);
    if (!c.ok) return;
    q_len[b] = c.q + c.blocks * kBlk;
    tail_len[b] = c.rest;
}

template <typename T>
static Buf<T> buf_of(const fg_kv8_cache* c, bool is_v) {
    return {(uint8_t*)(is_v ? c->v8 : c->k8), is_v ? c->v_scale : c->k_scale, (T*)(is_v ? c->v_tail : c->k_tail),
            c->batch, c->n_kv_heads, c->head_dim, c->capacity, c->tail_capacity};
}

// Shape and alignment of a cache; FG_OK when the kernels can run on it.
static fg_status check_cache(const fg_kv8_cache* c, int32_t B) {
    if (!c || !c->k8 || !c->v8 || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || c->n_layers <= 0 ||
        c->batch <= 0 || c->n_kv_heads <= 0 || c->capacity <= 0 || c->tail_capacity < kBlk || B < 0)
        return FG_EINVAL;
    if (c->dtype != FG_DTYPE_BF16 && c->dtype != FG_DTYPE_F32) return FG_EUNSUPPORTED;
    if (c->head_dim <= 0 || c->head_dim > kMaxD || c->head_dim % 16 || c->capacity % kBlk) return FG_EUNSUPPORTED;
    if (((uintptr_t)c->k8 | (uintptr_t)c->v8 | (uintptr_t)c->k_tail | (uintptr_t)c->v_tail) % 16) return FG_EINVAL;
    if (!c->rows && B > c->batch) return FG_EINVAL;
    // grid limits of the kernels' y and z
    if (B > 65535 || c->n_kv_heads > 16384 || c->n_layers > 65535) return FG_ECAPACITY;
    return FG_OK;
}

// Whether two int32 arrays share memory (NULL shares with none): lengths that
// a kernel writes while other CTAs still read them as something else.
static bool overlap(const int32_t* a, int64_t na, const int32_t* b, int64_t nb) {
    return a && b && (uintptr_t)a < (uintptr_t)(b + nb) && (uintptr_t)b < (uintptr_t)(a + na);
}

}  // namespace kv8
}  // namespace fg

using namespace fg;

extern "C" fg_status fg_kv8_load(const fg_kv8_cache* cache, int32_t layer, const void* k, const void* v,
                                 int64_t stride_b, int64_t stride_h, int64_t stride_s, int32_t src_len,
                                 const int32_t* lengths, int32_t n_src, int32_t repeats, int32_t* q_len,
                                 int32_t* tail_len, void* stream) {
    if (n_src < 0 || repeats <= 0 || (int64_t)n_src * repeats > 65535) return FG_EINVAL;
    const fg_status s = kv8::check_cache(cache, n_src * repeats);
    if (s != FG_OK) return s;
    if (n_src == 0) return FG_OK;
    if (layer < 0 || layer >= cache->n_layers || src_len < 0 || (src_len > 0 && (!k || !v)) || !lengths || !q_len ||
        !tail_len || q_len == tail_len)
        return FG_EINVAL;
    if (src_len / kv8::kBlk * kv8::kBlk > cache->capacity) return FG_ECAPACITY;
    const int64_t n = (int64_t)n_src * repeats;
    if (kv8::overlap(q_len, n, tail_len, n)) return FG_EINVAL;
    for (const int32_t* out : {q_len, tail_len})
        if (kv8::overlap(out, n, lengths, n_src) || kv8::overlap(out, n, cache->rows, n)) return FG_EINVAL;
    const int esz = cache->dtype == FG_DTYPE_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) % 16 == 0) && (stride_b * esz) % 16 == 0 &&
                     (stride_h * esz) % 16 == 0 && (stride_s * esz) % 16 == 0;
    const dim3 grid(src_len / kv8::kBlk + 1, 2 * cache->n_kv_heads, n_src);
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dtype == FG_DTYPE_F32)
        kv8::load_kernel<float><<<grid, kv8::kNT, 0, st>>>(
            kv8::buf_of<float>(cache, false), kv8::buf_of<float>(cache, true), layer, (const float*)k,
            (const float*)v, stride_b, stride_h, stride_s, vec, src_len, lengths, repeats, cache->rows, q_len,
            tail_len);
    else
        kv8::load_kernel<__nv_bfloat16><<<grid, kv8::kNT, 0, st>>>(
            kv8::buf_of<__nv_bfloat16>(cache, false), kv8::buf_of<__nv_bfloat16>(cache, true), layer,
            (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, stride_b, stride_h, stride_s, vec, src_len, lengths,
            repeats, cache->rows, q_len, tail_len);
    return launch_status();
}

extern "C" fg_status fg_kv8_commit(const fg_kv8_cache* cache, const int32_t* acc_nodes, int32_t dcap,
                                   const int32_t* acc_len, int32_t B, int32_t* q_len, int32_t* tail_len,
                                   int32_t* q_len_out, int32_t* tail_len_out, void* stream) {
    const fg_status s = kv8::check_cache(cache, B);
    if (s != FG_OK) return s;
    if (B == 0) return FG_OK;
    if (!acc_nodes || !acc_len || !q_len || !tail_len || q_len == tail_len || dcap <= 0 || !q_len_out != !tail_len_out) return FG_EINVAL;
    if (dcap > FG_MAX_PATH) return FG_ECAPACITY;
    if (q_len_out == q_len && tail_len_out == tail_len) q_len_out = tail_len_out = nullptr;  // in place
    // lengths, paths and rows that some CTAs still read must not change under them
    if (kv8::overlap(q_len, B, tail_len, B) || kv8::overlap(q_len_out, B, tail_len_out, B)) return FG_EINVAL;
    for (const int32_t* out : {q_len_out, tail_len_out})
        if (kv8::overlap(out, B, q_len, B) || kv8::overlap(out, B, tail_len, B)) return FG_EINVAL;
    for (const int32_t* out : {q_len_out ? q_len_out : q_len, q_len_out ? tail_len_out : tail_len})
        if (kv8::overlap(out, B, acc_len, B) || kv8::overlap(out, B, acc_nodes, (int64_t)B * dcap) ||
            kv8::overlap(out, B, cache->rows, B))
            return FG_EINVAL;
    const dim3 grid(2 * cache->n_kv_heads, cache->n_layers, B);
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dtype == FG_DTYPE_F32)
        kv8::commit_kernel<float><<<grid, kv8::kNT, 0, st>>>(
            kv8::buf_of<float>(cache, false), kv8::buf_of<float>(cache, true), acc_nodes, dcap, acc_len, cache->rows,
            q_len, tail_len, q_len_out, tail_len_out);
    else
        kv8::commit_kernel<__nv_bfloat16><<<grid, kv8::kNT, 0, st>>>(
            kv8::buf_of<__nv_bfloat16>(cache, false), kv8::buf_of<__nv_bfloat16>(cache, true), acc_nodes, dcap,
            acc_len, cache->rows, q_len, tail_len, q_len_out, tail_len_out);
    if (!q_len_out)
        kv8::commit_lengths_kernel<<<(B + 127) / 128, 128, 0, st>>>(acc_nodes, dcap, acc_len, cache->rows,
                                                                    cache->batch, cache->capacity,
                                                                    cache->tail_capacity, B, q_len, tail_len);
    return launch_status();
}
