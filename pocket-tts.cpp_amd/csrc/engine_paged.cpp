// LM state whose keys and values live in a pool of pages (ptts_state_new_paged): slots share one pool instead of holding a cache of
// fixed length each, may share the pages of a common prefix (one voice, many utterances), and with a window give back the pages
// that have fallen behind it, so that a stream of any length runs in a bounded pool.
//
// The host deals the pages out (it knows every slot's length); the GPU enters them in the block table and derives slot maps and
// positions with ptts_paged_plan, and every layer runs ptts_rotary_append and ptts_paged_attention in the place of the fixed
// cache's rotate / append and attention kernels.
#include <algorithm>
#include <cmath>

#include "engine.h"
#include "paged.h"
#include "rotary_frequencies.h"

namespace ptts {

// Sinks beyond the context are the whole context; as such their page count stays inside an int.
static PagedOptions within(PagedOptions o) {
    o.sinks = std::min(o.sinks, o.max_context);
    return o;
}

PagedCache::PagedCache(const Spec& s, int slots, int kv16_, const PagedOptions& o) : opt(within(o)), kv16(kv16_), layers(s.lm_layers), heads(s.lm_heads) {
    if (slots <= 0 || o.pages <= 0 || o.page_size <= 0 || o.max_context <= 0) throw std::runtime_error("slots, pages, page_size and max_context must be positive");
    if (static_cast<long long>(o.pages) * o.page_size >= 1ll << 30 || o.max_context >= 1 << 30) throw std::runtime_error("the pool must hold fewer than 2^30 rows");
    if (o.window < 0 || o.sinks < 0) throw std::runtime_error("window and sinks must not be negative");
    if (s.d_model != s.lm_heads * 64) throw std::runtime_error("head dimension must be 64");
    width = (o.max_context + o.page_size - 1) / o.page_size;
    if (static_cast<long long>(width) * o.page_size >= 1ll << 30) throw std::runtime_error("max_context is too long for this page size");
    layer_bytes = static_cast<size_t>(o.pages) * o.page_size * s.d_model * (kv16 ? 2 : 4);
    k.alloc(layer_bytes * layers);
    v.alloc(layer_bytes * layers);
    table.alloc(static_cast<size_t>(slots) * width * 4);
    ints.alloc((static_cast<size_t>(5) * slots + 2) * 4 + static_cast<size_t>(o.pages) * 4 + 64);
    // inputs of the plan: cached [slots], arriving [slots], fresh pages [pages]; its outputs: cu_rows [slots + 1], kv_len [slots], counts [4], status
    cached = ints.as<int>();
    arriving = cached + slots;
    fresh = arriving + slots;
    cu = fresh + o.pages;
    kv_len = cu + slots + 1;
    counts = kv_len + slots;
    status = counts + 4;
    std::vector<double> f(32);
    rotary_frequencies(64, s.lm_max_period, 0, 1.0, 0.0, 0.0, 0.0, f.data(), nullptr);
    freq.alloc(f.size() * 8);
    sync_copy(freq.p, f.data(), f.size() * 8, hipMemcpyHostToDevice);
    PTTS_HIP(hipHostMalloc(reinterpret_cast<void**>(&host), (2 * static_cast<size_t>(slots) + o.pages) * 4));
    held.resize(slots);
    uses.assign(o.pages, 0);
    clear();
}

PagedCache::~PagedCache() {
    if (host) (void)hipHostFree(host);
}

void PagedCache::clear() {
    for (auto& h : held) h.clear();
    std::fill(uses.begin(), uses.end(), 0);
    free_pages.resize(opt.pages);
    for (int i = 0; i < opt.pages; ++i) free_pages[i] = opt.pages - 1 - i;      // taken from the back: page 0 first
    sync_fill(table.p, 0xff, table.bytes);
    sync_fill(status, 0, 4);
}

void PagedCache::release(int page) {
    if (page >= 0 && --uses[page] == 0) free_pages.push_back(page);
}

// Pages of a slot that no row from position `length` on can see: behind the window and past the sinks.
template <typename F> void PagedCache::behind_window(int slot, int length, F&& take) {
    if (opt.window == 0) return;
    const long long low = static_cast<long long>(length) - opt.window + 1;      // first key that the next row's window holds
    auto& h = held[slot];
    for (long long i = (opt.sinks + opt.page_size - 1) / opt.page_size; i < static_cast<long long>(h.size()) && (i + 1) * opt.page_size <= low; ++i)
        if (h[i] >= 0) take(h[i]);
}

// Throws if `rows` new rows of a slot, taken `chunk` at a time, would run out of pages or of context; changes nothing.
void PagedCache::check_room(int slot, int length, int rows, int chunk) const {
    if (length + static_cast<long long>(rows) > opt.max_context) throw std::runtime_error("LM context exceeds max_context");
    long long free = free_count(), have = static_cast<long long>(held[slot].size()), dead = (opt.sinks + opt.page_size - 1) / opt.page_size;
    while (dead < have && held[slot][dead] < 0) ++dead;
    for (int done = 0; done < rows; done += chunk) {
        const long long low = opt.window ? static_cast<long long>(length) + done - opt.window + 1 : 0, n = std::min(chunk, rows - done);
        for (; dead < have && (dead + 1) * opt.page_size <= low; ++dead) free += dead >= static_cast<long long>(held[slot].size()) || uses[held[slot][dead]] == 1;
        const long long need = std::max(0ll, pages_of(length + done + n) - have);
        if (need > free) throw std::runtime_error("the pool has " + std::to_string(free_pages.size()) + " free pages, too few for " + std::to_string(rows) + " rows");
        free -= need;
        have += need;
    }
}

// Block table, slot map and positions of `rows` new rows of each slot slot0 .. slot0 + nb - 1, at the lengths `pos`.  Throws if they do
// not fit, before anything changes.
void PagedCache::plan(int slot0, int nb, int rows, const int* pos, hipStream_t st) {
    long long need = 0, back = 0;              // pages taken; pages that come back, those shared between these slots once
    for (int i = 0; i < nb; ++i) {
        if (pos[i] + static_cast<long long>(rows) > opt.max_context) throw std::runtime_error("LM context exceeds max_context");
        need += std::max(0ll, pages_of(pos[i] + rows) - static_cast<long long>(held[slot0 + i].size()));
    }
    for (int i = 0; i < nb; ++i) behind_window(slot0 + i, pos[i], [&](int page) { back += --uses[page] == 0; });
    for (int i = 0; i < nb; ++i) behind_window(slot0 + i, pos[i], [&](int page) { ++uses[page]; });
    if (need > free_count() + back)
        throw std::runtime_error("the pool has " + std::to_string(free_pages.size()) + " free pages, " + std::to_string(need) + " are needed");
    for (DevBuf* b : {&slot_map, &positions})
        if (b->bytes < static_cast<size_t>(nb) * rows * 4) {
            PTTS_HIP(hipStreamSynchronize(st));
            b->alloc(static_cast<size_t>(nb) * rows * 4);
        }
    PTTS_HIP(hipStreamSynchronize(st));        // the last call's copies have left the pinned block
    for (int i = 0; i < nb; ++i)
        behind_window(slot0 + i, pos[i], [&](int& page) {
            release(page);
            page = -1;
        });
    int taken = 0;
    most = 0;
    for (int i = 0; i < nb; ++i) {
        host[i] = pos[i];
        host[nb + i] = rows;
        most = std::max(most, pos[i] + rows);
        // The plan is given every page behind the slot's rows, those too that a call which failed after its plan has left here.
        auto& h = held[slot0 + i];
        const long long last = pages_of(pos[i] + rows);
        while (static_cast<long long>(h.size()) < last) {
            const int page = free_pages.back();
            free_pages.pop_back();
            uses[page] = 1;
            h.push_back(page);
        }
        for (long long k = pages_of(pos[i]); k < last; ++k) host[2 * nb + taken++] = h[k];
    }
    PTTS_HIP(hipMemcpyAsync(cached, host, static_cast<size_t>(nb) * 4, hipMemcpyHostToDevice, st));
    PTTS_HIP(hipMemcpyAsync(arriving, host + nb, static_cast<size_t>(nb) * 4, hipMemcpyHostToDevice, st));
    if (taken) PTTS_HIP(hipMemcpyAsync(fresh, host + 2 * nb, static_cast<size_t>(taken) * 4, hipMemcpyHostToDevice, st));
    PttsPagedPlan p{};
    p.cached = cached; p.arriving = arriving; p.free_pages = fresh; p.n_free = taken;
    p.block_table = table.as<int>() + static_cast<size_t>(slot0) * width; p.table_stride = width; p.table_width = width;
    p.slot_map = slot_map.as<int>(); p.positions = positions.as<int>(); p.cu_rows = cu; p.kv_len = kv_len; p.counts = counts; p.status = status;
    p.requests = nb; p.page_size = opt.page_size; p.rows = nb * rows;
    check_paged_plan(p);
    launch_paged_plan(p, st);
    now_slot0 = slot0; now_nb = nb; now_rows = rows;
}

// One layer's rows qkv[nb * rows][3 d]: rotated, filed, attended.  q: scratch rows, out: attention output, both [nb * rows][d] f32.
void PagedCache::attend(int layer, const float* qkv, int d, float* q, float* out, int cus, hipStream_t st) {
    const int M = now_nb * now_rows;
    PttsPages pages{};
    pages.k = k.as<char>() + layer_bytes * layer;
    pages.v = v.as<char>() + layer_bytes * layer;
    pages.type = kv16 ? PTTS_TYPE_BF16 : PTTS_TYPE_F32;
    pages.pages = opt.pages; pages.page_size = opt.page_size; pages.kv_heads = heads; pages.head_dim = 64;
    pages.page_stride = static_cast<long long>(opt.page_size) * d; pages.row_stride = d; pages.head_stride = 64;
    PttsRotaryAppend r{};
    r.q = qkv; r.k = qkv + d; r.v = qkv + 2 * d; r.q_out = q;
    r.q_row_stride = r.k_row_stride = r.v_row_stride = 3ll * d; r.q_head_stride = r.k_head_stride = r.v_head_stride = 64;
    r.out_row_stride = d; r.out_head_stride = 64;
    r.positions = positions.as<int>(); r.slot_map = slot_map.as<int>(); r.freq = freq.as<double>(); r.status = status;
    r.pages = pages; r.magnitude = 1.0f; r.type = PTTS_TYPE_F32; r.rows = M; r.q_heads = heads; r.rot_dim = 64; r.interleaved = 1;
    check_rotary_append(r);
    launch_rotary_append(r, st);
    PttsPagedAttention a{};
    a.q = q; a.out = out; a.cu_rows = cu; a.kv_len = kv_len; a.block_table = table.as<int>() + static_cast<size_t>(now_slot0) * width; a.status = status;
    a.q_row_stride = a.out_row_stride = d; a.q_head_stride = a.out_head_stride = 64; a.table_stride = width;
    a.pages = pages; a.scale = 0.125f; a.q_type = PTTS_TYPE_F32; a.rows = M; a.requests = now_nb; a.q_heads = heads; a.table_width = width;
    a.window = opt.window; a.sinks = opt.sinks; a.max_rows = now_rows; a.max_kv = most;
    check_paged_attention(a);
    const long long need = paged_attention_workspace(a, cus);
    if (static_cast<size_t>(need) > work.bytes) {
        PTTS_HIP(hipStreamSynchronize(st));
        work.alloc(static_cast<size_t>(need));
    }
    a.workspace = work.p;
    a.workspace_bytes = static_cast<long long>(work.bytes);
    launch_paged_attention(a, cus, st);
}

// The first `rows` rows of slot `from` become slot `to`'s: whole pages are shared, the rows of a last page that is partly filled are copied
// (rows would be appended to it).
void PagedCache::share(int from, int to, int rows, int from_length, hipStream_t st) {
    const int slots = static_cast<int>(held.size());
    if (from < 0 || from >= slots || to < 0 || to >= slots || from == to) throw std::runtime_error("two slots of the state are required");
    if (rows < 0 || rows > from_length) throw std::runtime_error("slot " + std::to_string(from) + " holds " + std::to_string(from_length) + " rows");
    const int whole = rows / opt.page_size, rest = rows % opt.page_size, used = whole + (rest ? 1 : 0);
    const auto& f = held[from];
    for (int i = 0; i < used; ++i)
        if (f[i] < 0) throw std::runtime_error("rows behind the window have been given back");
    const bool own = std::any_of(held[to].begin(), held[to].end(), [&](int page) { return page >= 0 && uses[page] == 1; });   // come back below
    if (rest && free_pages.empty() && !own) throw std::runtime_error("the pool has no free page");
    drop(to);
    auto& t = held[to];
    t.assign(f.begin(), f.begin() + whole);
    for (int page : t) ++uses[page];
    if (rest) {
        const int page = free_pages.back();
        free_pages.pop_back();
        uses[page] = 1;
        t.push_back(page);
        const size_t row = layer_bytes / (static_cast<size_t>(opt.pages) * opt.page_size), stride = row * opt.page_size;
        for (int l = 0; l < layers; ++l)
            for (DevBuf* b : {&k, &v})
                PTTS_HIP(hipMemcpyAsync(b->as<char>() + layer_bytes * l + stride * page, b->as<char>() + layer_bytes * l + stride * f[whole], row * rest,
                                        hipMemcpyDeviceToDevice, st));
    }
    if (used) PTTS_HIP(hipMemcpyAsync(table.as<int>() + static_cast<size_t>(to) * width, t.data(), static_cast<size_t>(used) * 4, hipMemcpyHostToDevice, st));
    PTTS_HIP(hipStreamSynchronize(st));
}

void PagedCache::drop(int slot) {
    for (int page : held[slot]) release(page);
    held[slot].clear();
}

// Bad page ids or lengths would be a mistake of the bookkeeping above: the kernels do not read them and say so here.
void PagedCache::check_status() {
    int s = 0;
    sync_copy(&s, status, 4, hipMemcpyDeviceToHost);
    if (s) throw std::runtime_error("the paged cache reports status " + std::to_string(s));
}

Batch* Engine::batch_new_paged(int B, const PagedOptions& o) {
    PTTS_HIP(hipSetDevice(opt_.device));
    return new Batch(*this, B, false, &o);
}

int Engine::op_state_free_pages(Batch* b) {
    std::lock_guard<std::mutex> guard(mu_);
    if (!b->paged) throw std::runtime_error("the state was not created with pages");
    return b->paged->free_count();
}

void Engine::op_state_share(Batch* b, int from, int to, int rows) {
    std::lock_guard<std::mutex> guard(mu_);
    PTTS_HIP(hipSetDevice(opt_.device));
    if (!b->paged) throw std::runtime_error("the state was not created with pages");
    const int length = from >= 0 && from < b->B ? b->lm_pos_host[from] : 0;
    b->paged->share(from, to, rows, length, b->st);
    b->lm_pos_host[to] = rows;
    PTTS_HIP(hipMemcpyAsync(b->lm_pos.as<int>() + to, &b->lm_pos_host[to], 4, hipMemcpyHostToDevice, b->st));
    PTTS_HIP(hipStreamSynchronize(b->st));
}

}  // namespace ptts
