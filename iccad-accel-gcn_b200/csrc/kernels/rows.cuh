// Rows of features in 32 or 16 bits, 16 bytes per thread at a time: what the layer norm and dropout kernels share.
//
// All of these kernels are launched early (programmatic dependent launch): their thread blocks get ready while the launch before
// them on the stream, whatever it is, comes to its end, and wait for it before they touch memory.  2 048 rows of 16 back to back:
// 2.6 us a launch in place of 3.9; 2 us less at every size.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace agcn {

// How the rows of all tensors of a call sit: alike with respect to 16-byte boundaries, every row beginning and ending on
// one (WHOLE); alike, with chunks at the rows' ends that are not the row's alone (EDGES); or not alike (LOOSE: read
// element by element).
enum RowLayout { ROWS_WHOLE, ROWS_EDGES, ROWS_LOOSE };

// E elements of type T are 16 bytes.  All arithmetic is in fp32; the one rounding to T is that of the result.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4 &r, float *v)
    {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4 &r, float *v)
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int k = 0; k < 4; k++) { v[2 * k] = __uint_as_float(w[k] << 16); v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Elem<__half> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4 &r, float *v)
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            v[2 * k] = f.x; v[2 * k + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *v)
    {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
            w[k] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Two fp32 operations in one instruction (both rounded as the single ones are): fewer instructions for the few warps that there are
// (2 400 000 x 128, layer norm: 435 -> 417 us, backward 650 -> 625-645).
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 pair(const float *v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ void unpair(float2 p, float *v) { v[0] = p.x; v[1] = p.y; }

// Columns c0 .. c0 + E - 1 of a row, as far as they are in [0, cols); zeros elsewhere.  VEC: a whole chunk is one access
// (column c0 then sits on a 16-byte boundary); the chunks at the ends of a row go element by element, so that nothing
// outside the row is touched.
template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T *row, int c0, int cols, float *v)
{
    constexpr int E = Elem<T>::E;
    if (VEC && c0 >= 0 && c0 + E <= cols) {
        Elem<T>::unpack(*reinterpret_cast<const uint4 *>(row + c0), v);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = c0 + e >= 0 && c0 + e < cols ? Elem<T>::get(row[c0 + e]) : 0.f;
    }
}
// The same into memory, to `to` on: the elements whose bits are set.  WHOLE: all of them are known to be.
template <typename T, bool VEC, bool WHOLE>
__device__ __forceinline__ void store_chunk(T *to, uint32_t bits, const float *v)
{
    constexpr int E = Elem<T>::E;
    if (VEC && (WHOLE || bits == (1u << E) - 1)) {
        *reinterpret_cast<uint4 *>(to) = Elem<T>::pack(v);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) if (bits >> e & 1u) to[e] = Elem<T>::put(v[e]);
    }
}

// 16 bytes from global to shared memory behind the thread's back; what is past `bytes` becomes 0 and is not read.
__device__ __forceinline__ void copy_chunk(uint32_t to, const void *from, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_chunk(uint32_t to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most N of the thread's groups of copies are under way
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ uint4 load_shared(uint32_t from)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared(uint32_t to, const uint4 &v)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" :: "r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A thread's ring of rows that are under way from memory: STAGES rows ahead, N tensors, CH chunks each.  A slot belongs to
// one thread, which fills and reads it: nothing to synchronise.  Registers hold the row that is worked on and nothing
// else, and the bytes in flight do not depend on how many threads fit an SM.
template <typename T, int N, int CH, int STAGES>
struct RowRing {
    uint32_t at, begin, slots;           // this thread's place in the stage that is read next, and in the first; bytes between two slots
    __device__ __forceinline__ RowRing(void *s) : at((uint32_t)__cvta_generic_to_shared(s) + threadIdx.x * 16u), begin(at), slots(blockDim.x * 16u) {}
    __device__ __forceinline__ uint32_t slot(int k, int j) const { return at + (k * CH + j) * slots; }
    __device__ __forceinline__ void next()
    {
        at += N * CH * slots;
        if (at == begin + STAGES * N * CH * slots) at = begin;
    }
    __device__ __forceinline__ void clear() const
    {
#pragma unroll
        for (int k = 0; k < N * CH; k++) store_shared(at + k * slots, make_uint4(0, 0, 0, 0));
    }
    // Starts the copy of chunk j of tensor k: of a whole one at `from`, ...
    __device__ __forceinline__ void fetch(int k, int j, const T *from) const { copy_chunk(slot(k, j), from); }
    // ... or of `bytes` of it: what is in front of the row within its first 16 bytes comes along, unused, ...
    __device__ __forceinline__ void fetch(int k, int j, const T *from, int bytes) const { copy_chunk(slot(k, j), from, bytes); }
    // ... but not where that would be in front of the tensor, at `first` (the chunk has elements c0 .. of a row; only the first few rows
    // can be that near).
    __device__ __forceinline__ void fetch_edge(int k, int j, const T *from, const T *first, int c0, int cols, int bytes) const
    {
        if (from < first) {
            float v[Elem<T>::E];
            load_chunk<T, false>(from - c0, c0, cols, v);
            store_shared(slot(k, j), Elem<T>::pack(v));
        } else {
            fetch(k, j, from, bytes);
        }
    }
    __device__ __forceinline__ uint4 get(int k, int j) const { return load_shared(slot(k, j)); }
    __device__ __forceinline__ void get(int k, int j, float *v) const { Elem<T>::unpack(get(k, j), v); }
};

__device__ __forceinline__ float masked(float v, uint32_t bits) { return __uint_as_float(__float_as_uint(v) & bits); }

// max(v, 0) that lets NaN through, and whether a gradient passes
__device__ __forceinline__ float relu_of(float v)
{
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ bool relu_passes(float v) { return !(v <= 0.f); }

// Sums of K values over a group of L lanes of a warp, or (L = 0) over the thread block; every thread gets them, added
// in one order.  All lanes of the warp (threads of the block) call.  s_sums: zero where there is no warp; `turn` says which half is
// free: the other one may still be read by warps that are behind.
constexpr int ROW_WARPS = 16;              // most warps of a thread block that has one row
template <int K> struct GroupSums { alignas(16) float v[2][K][ROW_WARPS]; };
template <int K>
__device__ __forceinline__ void clear_sums(GroupSums<K> &s)
{
    for (int i = threadIdx.x; i < 2 * K * ROW_WARPS; i += blockDim.x) (&s.v[0][0][0])[i] = 0.f;
}
template <int L, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], GroupSums<K> &s_sums, int &turn)
{
    static_assert(K == 1 || K == 2, "");
    if (L > 0) {
#pragma unroll
        for (int d = L / 2; d > 0; d >>= 1) {
#pragma unroll
            for (int k = 0; k < K; k++) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
        }
    } else {
        // Half of the lanes add up one value and half the other: one exchange more than for one value, not five.
        const int lane = threadIdx.x & 31;
        float s = v[0];
        if (K == 2) s = (lane & 16 ? v[K - 1] : v[0]) + __shfl_xor_sync(0xffffffffu, lane & 16 ? v[0] : v[K - 1], 16);
        else s += __shfl_xor_sync(0xffffffffu, s, 16);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if ((lane & 15) == 0) s_sums.v[turn][K == 2 ? lane >> 4 : 0][threadIdx.x >> 5] = s;
        __syncthreads();
        s = s_sums.v[turn][K == 2 ? lane >> 4 : 0][lane & 15];
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        v[0] = s;
        if (K == 2) {
            const float other = __shfl_xor_sync(0xffffffffu, s, 16);
            v[0] = lane & 16 ? other : s;
            v[K - 1] = lane & 16 ? s : other;
        }
        turn ^= 1;
    }
}

}  // namespace agcn
