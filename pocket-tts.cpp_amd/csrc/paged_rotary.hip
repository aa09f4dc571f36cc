// Rotary positions of the new rows, with their keys and values filed into the pages (pocket_tts_amd.h, ptts_rotary_append).
//
// (a, b) -> (a cos - b sin, b cos + a sin) for each pair of a head.  The angle positions[row] * freq[i] is formed in float64 and
// reduced to a fraction of a turn there, so that a position of a million loses nothing; sine and cosine of the fraction are
// float32.  They depend on (row, pair) alone: a workgroup computes them once for its row into LDS and then streams all heads past
// them, which leaves the kernel at one read and one write of q, k and v, its bound: 8192 rows of 32 / 8 heads of 128 in bf16 move 201 MB in
// 34.2 us, 5.9 TB/s (a large copy reaches 5.1); 1001 rows of 12 / 4 heads of 96 take 4.1 us, 64 rows of 16 heads 4.1, a launch's own time.
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "paged.h"

namespace ptts {

namespace {

struct RotaryArgs {
    PttsRotaryAppend p;
    FastDiv page;
    int units;       // work units of one row: rotated heads (q, k) times units per head, then v
    FastDiv per_head, per_v;   // units of a rotated head, of a value head
};

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

// N values: one access, or value by value for the narrow form, which makes no demand on alignment.  kStream: past the caches.
template <typename T, int N, bool kStream> __device__ __forceinline__ void load_f(const T* p, float* x) {
    if constexpr (N <= 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)p[i];
    } else {
        typedef unsigned words __attribute__((ext_vector_type(sizeof(T) * N / 4)));
        union { words w; Vec<T, N> v; } u;
        if constexpr (kStream) u.w = __builtin_nontemporal_load(reinterpret_cast<const words*>(p));
        else u.w = *reinterpret_cast<const words*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)u.v.v[i];
    }
}
template <typename T, int N, bool kStream> __device__ __forceinline__ void store_f(T* p, const float* x) {
    if constexpr (N <= 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = (T)x[i];
    } else {
        typedef unsigned words __attribute__((ext_vector_type(sizeof(T) * N / 4)));
        union { words w; Vec<T, N> v; } u;
#pragma unroll
        for (int i = 0; i < N; ++i) u.v.v[i] = (T)x[i];
        if constexpr (kStream) __builtin_nontemporal_store(u.w, reinterpret_cast<words*>(p));
        else *reinterpret_cast<words*>(p) = u.w;
    }
}

// N values at a time (1: any alignment and any rot_dim).  Halves layout: a unit of the rotated part is N values of the first half and
// their partners in the second.  Interleaved: a unit is N (at least 2) neighbouring values, N / 2 pairs.
template <typename T, typename C, int N, bool INTER, bool kStream>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 turn[128];                         // [rot_dim / 2]
    __shared__ long long place;                          // element offset of the row's slot in the pages, -1: none
    const PttsRotaryAppend& p = a.p;
    const int tid = threadIdx.x, half = p.rot_dim >> 1;
    const int row = blockIdx.x;
    if (tid == 0) {
        long long at = -1;
        if (p.k) {
            const int slot = p.slot_map[row];
            const unsigned pg = slot < 0 ? 0 : a.page.div(slot);
            if (slot >= 0 && pg < (unsigned)p.pages.pages)
                at = (long long)pg * p.pages.page_stride + (long long)(slot - (int)pg * p.pages.page_size) * p.pages.row_stride;
            else if (slot != -1 && p.status) atomicOr(p.status, kStatusPage);
        }
        place = at;
    }
    if (tid < half) {
        const double t = (double)p.positions[row] * (p.freq[tid] * 0.15915494309189533577);   // turns
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        turn[tid] = make_float2(c * p.magnitude, s * p.magnitude);
    }
    __syncthreads();
    constexpr int NN = INTER && N == 1 ? 2 : N;          // values of a unit outside the halves layout
    const int rot_heads = (p.q ? p.q_heads : 0) + (p.k ? p.pages.kv_heads : 0), q_heads = p.q ? p.q_heads : 0;
    const int turn_units = INTER ? p.rot_dim / NN : half / N;
    const long long filed = place;
    for (int u = blockIdx.y * 256 + tid; u < a.units; u += gridDim.y * 256) {
        int w = u;
        const int n_rot = rot_heads * (int)a.per_head.d;
        if (w < n_rot) {
            const int h = (int)a.per_head.div(w), e = w - h * (int)a.per_head.d;
            const bool is_q = h < q_heads;
            if (!is_q && filed < 0) continue;
            const T* src = is_q ? (const T*)p.q + (long long)row * p.q_row_stride + (long long)h * p.q_head_stride
                                : (const T*)p.k + (long long)row * p.k_row_stride + (long long)(h - q_heads) * p.k_head_stride;
            T* qd = (T*)p.q_out + (long long)row * p.out_row_stride + (long long)h * p.out_head_stride;
            C* kd = is_q ? nullptr : (C*)p.pages.k + filed + (long long)(h - q_heads) * p.pages.head_stride;
            if (e >= turn_units) {                       // behind the rotated part
                const int d0 = p.rot_dim + (e - turn_units) * NN;
                float x[NN];
                load_f<T, NN, kStream>(src + d0, x);
                if (is_q) store_f<T, NN, kStream>(qd + d0, x);
                else store_f<C, NN, kStream>(kd + d0, x);
            } else if constexpr (INTER) {
                const int d0 = e * NN;
                float x[NN], y[NN];
                load_f<T, NN, kStream>(src + d0, x);
#pragma unroll
                for (int i = 0; i < NN / 2; ++i) {
                    const float2 cs = turn[d0 / 2 + i];
                    y[2 * i] = x[2 * i] * cs.x - x[2 * i + 1] * cs.y;
                    y[2 * i + 1] = x[2 * i + 1] * cs.x + x[2 * i] * cs.y;
                }
                if (is_q) store_f<T, NN, kStream>(qd + d0, y);
                else store_f<C, NN, kStream>(kd + d0, y);
            } else {
                const int d0 = e * N;
                float x0[N], x1[N], y0[N], y1[N];
                load_f<T, N, kStream>(src + d0, x0);
                load_f<T, N, kStream>(src + half + d0, x1);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float2 cs = turn[d0 + i];
                    y0[i] = x0[i] * cs.x - x1[i] * cs.y;
                    y1[i] = x1[i] * cs.x + x0[i] * cs.y;
                }
                if (is_q) { store_f<T, N, kStream>(qd + d0, y0); store_f<T, N, kStream>(qd + half + d0, y1); }
                else { store_f<C, N, kStream>(kd + d0, y0); store_f<C, N, kStream>(kd + half + d0, y1); }
            }
        } else {
            w -= n_rot;
            const int h = (int)a.per_v.div(w), d0 = (w - h * (int)a.per_v.d) * NN;
            if (filed < 0) continue;
            float x[NN];
            load_f<T, NN, kStream>((const T*)p.v + (long long)row * p.v_row_stride + (long long)h * p.v_head_stride + d0, x);
            store_f<C, NN, kStream>((C*)p.pages.v + filed + (long long)h * p.pages.head_stride + d0, x);
        }
    }
}

template <typename T, typename C>
void dispatch(RotaryArgs a, bool wide, hipStream_t s) {
    const PttsRotaryAppend& p = a.p;
    constexpr int W = 16 / sizeof(T);
    const int half = p.rot_dim / 2, nn = wide ? W : p.interleaved ? 2 : 1;
    const int per_head = (p.interleaved ? p.rot_dim / nn : half / (wide ? W : 1)) + (p.pages.head_dim - p.rot_dim) / nn;
    const int per_v = p.pages.head_dim / nn;
    const int rot_heads = (p.q ? p.q_heads : 0) + (p.k ? p.pages.kv_heads : 0);
    a.per_head = FastDiv::of(static_cast<unsigned>(per_head));
    a.per_v = FastDiv::of(static_cast<unsigned>(per_v));
    a.units = rot_heads * per_head + (p.k ? p.pages.kv_heads * per_v : 0);
    // One row a workgroup (two took 37.9 us in place of 34.6 for the 8192 rows below), and up to four workgroups a row where rows are few.
    const dim3 grid(p.rows, std::min(4, std::max(1, 256 / p.rows)));
    // What is more than the L2 caches hold between them (8 x 4 MB) cannot wait there for its reader, and passing it through them costs:
    // 8192 rows of 48 heads of 128 in bf16 (201 MB) take 41.9 us through the caches and 34.6 us past them (5.8 TB/s).  Smaller calls stay in
    // the caches, where the attention that follows finds them.
    const long long moved = static_cast<long long>(p.rows) * p.pages.head_dim * ((p.q ? 2ll * p.q_heads * sizeof(T) : 0) + (p.k ? 2ll * p.pages.kv_heads * (sizeof(T) + sizeof(C)) : 0));
    const bool stream = moved > 32ll << 20;
    if (wide) {
        if (p.interleaved && stream) launch_paged(rotary_kernel<T, C, W, true, true>, grid, s, a);
        else if (p.interleaved) launch_paged(rotary_kernel<T, C, W, true, false>, grid, s, a);
        else if (stream) launch_paged(rotary_kernel<T, C, W, false, true>, grid, s, a);
        else launch_paged(rotary_kernel<T, C, W, false, false>, grid, s, a);
    } else {
        if (p.interleaved) launch_paged(rotary_kernel<T, C, 1, true, false>, grid, s, a);
        else launch_paged(rotary_kernel<T, C, 1, false, false>, grid, s, a);
    }
}

uintptr_t low_bits(const PttsRotaryAppend& p) {
    uintptr_t low = 0;
    if (p.q) low |= reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.q_out);
    if (p.k) low |= reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    return low;
}

}  // namespace

void check_pages(const PttsPages& p, const char* who) {
    const std::string w = std::string(who) + ": ";
    if (!p.k || !p.v) throw std::runtime_error(w + "the pages need k and v");
    if (p.type != PTTS_TYPE_F32 && p.type != PTTS_TYPE_BF16 && p.type != PTTS_TYPE_F16) throw std::runtime_error(w + "unknown page type");
    if (p.pages < 1 || p.page_size < 1 || static_cast<long long>(p.pages) * p.page_size >= 1ll << 30)
        throw std::runtime_error(w + "pages and page_size must be positive and hold fewer than 2^30 rows");
    if (p.kv_heads < 1 || p.kv_heads > 65535) throw std::runtime_error(w + "kv_heads must be 1 to 65535");
    if (p.head_dim < 8 || p.head_dim > 256 || p.head_dim % 8) throw std::runtime_error(w + "head_dim must be a multiple of 8 up to 256");
    const int e = 16 / type_size(p.type);
    if (reinterpret_cast<uintptr_t>(p.k) % 16 || reinterpret_cast<uintptr_t>(p.v) % 16 || p.page_stride % e || p.row_stride % e || p.head_stride % e)
        throw std::runtime_error(w + "pages must be aligned to 16 bytes, strides too");
    if (p.page_stride < 0 || p.row_stride < 0 || p.head_stride < 0) throw std::runtime_error(w + "page strides must not be negative");
}

void check_rotary_append(const PttsRotaryAppend& p) {
    const char* who = "rotary_append";
    const std::string w = std::string(who) + ": ";
    if (p.rows < 0 || p.rows >= 1 << 24) throw std::runtime_error(w + "rows must be 0 to 2^24 - 1");
    if (p.rows > 0 && !p.q && !p.k) throw std::runtime_error(w + "nothing to rotate: q and k are both missing");
    if (!p.k != !p.v) throw std::runtime_error(w + "k and v come together");
    if (p.type != PTTS_TYPE_F32 && p.type != PTTS_TYPE_BF16 && p.type != PTTS_TYPE_F16) throw std::runtime_error(w + "unknown type");
    if (p.k) {
        check_pages(p.pages, who);
        if (p.pages.type != p.type && !(p.type == PTTS_TYPE_F32 && p.pages.type == PTTS_TYPE_BF16))
            throw std::runtime_error(w + "pages must have the rows' type, or bf16 under f32 rows");
    } else if (p.pages.head_dim < 8 || p.pages.head_dim > 256 || p.pages.head_dim % 8) {
        throw std::runtime_error(w + "head_dim must be a multiple of 8 up to 256");
    }
    if (p.q && (p.q_heads < 1 || p.q_heads > 65535)) throw std::runtime_error(w + "q_heads must be 1 to 65535");
    if (p.rot_dim < 2 || p.rot_dim % 2 || p.rot_dim > p.pages.head_dim) throw std::runtime_error(w + "rot_dim must be even, at least 2 and at most head_dim");
    if (!std::isfinite(p.magnitude)) throw std::runtime_error(w + "magnitude must be finite");
    if (p.rows == 0) return;
    if (!p.positions || !p.freq) throw std::runtime_error(w + "positions and freq are required");
    if (p.q && !p.q_out) throw std::runtime_error(w + "q_out is required");
    if (p.k && !p.slot_map) throw std::runtime_error(w + "slot_map is required");
    if (p.q == p.q_out && p.q && (p.q_row_stride != p.out_row_stride || p.q_head_stride != p.out_head_stride))
        throw std::runtime_error(w + "q_out may be q itself only with the same strides");
    if (!aligned({p.positions, p.slot_map, p.status}, 4) || !aligned({p.freq}, 8))
        throw std::runtime_error(w + "positions, slot_map and status must be aligned to 4 bytes, freq to 8");
    if (low_bits(p) % type_size(p.type)) throw std::runtime_error(w + "rows must be aligned to their type");
}

void launch_rotary_append(const PttsRotaryAppend& p, hipStream_t s) {
    if (p.rows == 0) return;
    // 16-byte accesses where every row of q, k, v and q_out allows them and no unit straddles the rotated part's borders;
    // else one value (pair) at a time.
    const int n = 16 / type_size(p.type), half = p.rot_dim / 2;
    long long str = 0;
    if (p.q) str |= p.q_row_stride | p.q_head_stride | p.out_row_stride | p.out_head_stride;
    if (p.k) str |= p.k_row_stride | p.k_head_stride | p.v_row_stride | p.v_head_stride;
    const bool wide = low_bits(p) % 16 == 0 && str % n == 0 && (p.interleaved ? p.rot_dim % n == 0 : half % n == 0) && (p.pages.head_dim - p.rot_dim) % n == 0;
    RotaryArgs a;
    a.p = p;
    a.page = FastDiv::of(static_cast<unsigned>(p.k ? p.pages.page_size : 1));
    if (p.type == PTTS_TYPE_F32 && p.k && p.pages.type == PTTS_TYPE_BF16) dispatch<float, __bf16>(a, wide, s);
    else if (p.type == PTTS_TYPE_F32) dispatch<float, float>(a, wide, s);
    else if (p.type == PTTS_TYPE_BF16) dispatch<__bf16, __bf16>(a, wide, s);
    else dispatch<_Float16, _Float16>(a, wide, s);
}

}  // namespace ptts
