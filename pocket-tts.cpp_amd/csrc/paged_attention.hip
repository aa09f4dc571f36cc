// Attention of every request's new rows over its pages (pocket_tts_amd.h, ptts_paged_attention).
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "paged.h"

namespace ptts {

namespace {

struct AttnArgs {
    PttsPagedAttention p;
    FastDiv page;
    int group;            // query heads per key head
    float scale2;         // scale * log2(e)
};

// The request that owns a row, or -1: the last i with cu_rows[i] <= row, found 64 requests at a time.
__device__ __forceinline__ int request_of_row(const PttsPagedAttention& p, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, span = p.requests;
    while (span > 1) {
        const int step = (span + 63) >> 6, i = lo + lane * step;
        const int hits = __popcll(__ballot(lane * step < span && p.cu_rows[i] <= row));
        if (hits == 0) return -1;
        const int left = span - (hits - 1) * step;
        lo += (hits - 1) * step;
        span = left < step ? left : step;
    }
    return p.cu_rows[lo] <= row && row < p.cu_rows[lo + 1] ? lo : -1;
}

// Plain form: one wave per (row, head), 64 keys at a time.  A lane forms the whole product of its own key with the query; the
// weighted sum walks the visible keys with the lanes on the head's values.
template <typename T, typename C>
__global__ __launch_bounds__(256) void attention_rows_kernel(AttnArgs a) {
    const PttsPagedAttention& p = a.p;
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = (int)(unit / p.q_heads), head = (int)(unit % p.q_heads);
    if (row >= p.rows) return;
    const int i = request_of_row(p, row);
    if (i < 0) return;
    const int r0 = p.cu_rows[i], r1 = p.cu_rows[i + 1];
    int len = p.kv_len[i], bad = 0;
    const long long cap = (long long)p.table_width * p.pages.page_size;
    if (r0 < 0 || r1 > p.rows) bad |= kStatusRows;
    if (len < 0) { len = 0; bad |= kStatusLength; }
    if (len > cap) { len = (int)cap; bad |= kStatusLength; }
    const int pos = len - (r1 - row);
    const int dim = p.pages.head_dim, kvh = head / a.group;
    const T* q = (const T*)p.q + (long long)row * p.q_row_stride + (long long)head * p.q_head_stride;
    const int* table = p.block_table + (long long)i * p.table_stride;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    int lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
    for (int k0 = 0; k0 <= pos; k0 += 64) {
        if (p.window > 0 && k0 >= p.sinks && k0 + 63 < lo) { k0 = lo / 64 * 64; }
        const int key = k0 + lane;
        bool see = key <= pos && (key >= lo || key < p.sinks);
        long long at = -1;
        if (see) {
            const int pg = (int)a.page.div(key), id = table[pg];
            if (id < 0 || id >= p.pages.pages) bad |= kStatusPage;
            else at = (long long)id * p.pages.page_stride + (long long)(key - pg * p.pages.page_size) * p.pages.row_stride + (long long)kvh * p.pages.head_stride;
        }
        float s = 0.f;
        if (at >= 0) for (int d = 0; d < dim; ++d) s += (float)q[d] * (float)((const C*)p.pages.k)[at + d];
        s = see ? s * a.scale2 : -INFINITY;
        float top = s;
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float mn = fmaxf(m, top);
        if (mn == -INFINITY) continue;
        const float w = see ? exp2f(s - mn) : 0.f, fade = exp2f(m - mn);
        float ws = w;
        for (int o = 32; o > 0; o >>= 1) ws += __shfl_xor(ws, o, 64);
        l = l * fade + ws;
        m = mn;
        for (int c = 0; c < 4; ++c) acc[c] *= fade;
        unsigned long long left = __ballot(at >= 0);
        while (left) {
            const int j = __builtin_ctzll(left);
            left &= left - 1;
            const float wj = __shfl(w, j, 64);
            const long long aj = __shfl(at, j, 64);
            for (int c = 0; c < 4; ++c)
                if (lane + 64 * c < dim) acc[c] += wj * (float)((const C*)p.pages.v)[aj + lane + 64 * c];
        }
    }
    if (bad && p.status) atomicOr(p.status, bad);
    T* out = (T*)p.out + (long long)row * p.out_row_stride + (long long)head * p.out_head_stride;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < dim) out[lane + 64 * c] = (T)(l == 0.f ? 0.f : acc[c] * inv);
    if (p.lse && lane == 0) p.lse[(long long)row * p.lse_row_stride + head] = l == 0.f ? -INFINITY : m * 0.69314718055994531f + logf(l);
}

}  // namespace

void check_paged_attention(const PttsPagedAttention& p) {
    const std::string w = "paged_attention: ";
    if (p.rows < 0 || p.rows >= 1 << 30) throw std::runtime_error(w + "rows must be 0 to 2^30 - 1");
    if (p.requests < 0 || p.requests > 65536) throw std::runtime_error(w + "requests must be 0 to 65536");
    check_pages(p.pages, "paged_attention");
    if (p.q_type != PTTS_TYPE_F32 && p.q_type != PTTS_TYPE_BF16 && p.q_type != PTTS_TYPE_F16) throw std::runtime_error(w + "unknown type");
    if (p.pages.type != p.q_type && !(p.q_type == PTTS_TYPE_F32 && p.pages.type == PTTS_TYPE_BF16))
        throw std::runtime_error(w + "pages must have the rows' type, or bf16 under f32 rows");
    if (p.q_heads < 1 || p.q_heads > 65535 || p.q_heads % p.pages.kv_heads) throw std::runtime_error(w + "q_heads must be a multiple of kv_heads, at most 65535");
    if (!(p.scale > 0.f) || !std::isfinite(p.scale)) throw std::runtime_error(w + "scale must be positive and finite");
    if (p.sinks < 0) throw std::runtime_error(w + "sinks must not be negative");
    if (p.max_rows < 0 || p.max_kv < 0) throw std::runtime_error(w + "max_rows and max_kv must not be negative");
    if (p.table_width < 0 || static_cast<long long>(p.table_width) * p.pages.page_size >= 1ll << 30)
        throw std::runtime_error(w + "table_width * page_size must be below 2^30");
    if (p.requests > 1 && p.table_stride < p.table_width) throw std::runtime_error(w + "table_stride is smaller than table_width");
    if (p.rows == 0 || p.requests == 0) return;
    if (!p.q || !p.out || !p.cu_rows || !p.kv_len || (p.table_width > 0 && !p.block_table))
        throw std::runtime_error(w + "q, out, cu_rows, kv_len and block_table are required");
    if (p.q == p.out) throw std::runtime_error(w + "out must not be q");
    const int e = 16 / type_size(p.q_type);
    if (reinterpret_cast<uintptr_t>(p.q) % 16 || p.q_row_stride % e || p.q_head_stride % e || reinterpret_cast<uintptr_t>(p.out) % 16 ||
        p.out_row_stride % e || p.out_head_stride % e)
        throw std::runtime_error(w + "q and out must be aligned to 16 bytes, strides too");
}

long long paged_attention_workspace(const PttsPagedAttention& p, int cus) {
    (void)cus;
    return 0;
}

void launch_paged_attention(const PttsPagedAttention& p, int cus, hipStream_t s) {
    (void)cus;
    if (p.rows == 0 || p.requests == 0) return;
    AttnArgs a;
    a.p = p;
    a.p.window = p.window > 1 << 30 ? 0 : p.window;   // no context is that long
    a.page = FastDiv::of(static_cast<unsigned>(p.pages.page_size));
    a.group = p.q_heads / p.pages.kv_heads;
    a.scale2 = p.scale * 1.4426950408889634f;
    const long long units = static_cast<long long>(p.rows) * p.q_heads;
    if ((units + 3) / 4 > 0x7fffffffll) throw std::runtime_error("paged_attention: too many rows and heads for one call");
    const dim3 grid(static_cast<unsigned>((units + 3) / 4)), block(256);
    if (p.q_type == PTTS_TYPE_F32 && p.pages.type == PTTS_TYPE_BF16) hipLaunchKernelGGL((attention_rows_kernel<float, __bf16>), grid, block, 0, s, a);
    else if (p.q_type == PTTS_TYPE_F32) hipLaunchKernelGGL((attention_rows_kernel<float, float>), grid, block, 0, s, a);
    else if (p.q_type == PTTS_TYPE_BF16) hipLaunchKernelGGL((attention_rows_kernel<__bf16, __bf16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attention_rows_kernel<_Float16, _Float16>), grid, block, 0, s, a);
}

}  // namespace ptts
