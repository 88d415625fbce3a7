// C ABI of the decode operators that stand beside the model: the 8-bit K/V cache with its attention
// and beam search's selection and reordering.  Declared in include/stt_b200.h.
#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

#include "beam.h"
#include "host_util.h"
#include "kv8.h"

using namespace stt;

struct stt_kv8_cache {
    int device = 0;
    Kv8Machine machine{};
    Kv8Dev c{};
    void* memory = nullptr;   // codes and exponents; the library's own unless the caller gave it
    bool owned = false;
    void* scratch = nullptr;  // error word, tickets, attention partials
    float* part = nullptr;
    uint32_t* tickets = nullptr;
};

struct stt_beam {
    int device = 0, num_sms = 0;
    int max_batch = 0, max_beams = 0, max_vocab = 0;
    void* scratch = nullptr;
    int32_t* err = nullptr;
    BeamArgs ws{};  // the workspace pointers
};

namespace {

int elem_bytes(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// Tiles of a row, which may start 7 elements into its first vector, and the most CTAs that share them.
int beam_tiles(int vocab, int dtype) { return (vocab + 7 + beam_tile(dtype) - 1) / beam_tile(dtype); }
int beam_max_chunks(int vocab, int dtype) { return std::min(kBeamMaxChunks, beam_tiles(vocab, dtype)); }

// n_seqs * heads * capacity * dim and the sizes derived from it; false if the arguments do not make a cache.
bool kv8_sizes(int n_seqs, int heads, int dim, int cap, size_t* codes, size_t* exps) {
    if (n_seqs <= 0 || heads <= 0 || (dim != 64 && dim != 128) || cap <= 0 || cap % kKv8Block != 0) return false;
    const unsigned __int128 slots = (unsigned __int128)n_seqs * heads * cap;
    if (slots * dim > (unsigned __int128)1 << 48) return false;
    *codes = (size_t)slots * dim;
    *exps = (size_t)slots / kKv8Block;
    return true;
}

Kv8Strides strides(const stt_kv8_tensor& t) { return Kv8Strides{t.seq_stride, t.token_stride, t.head_stride}; }

int check_tensor(const char* what, const stt_kv8_tensor& t) {
    if (t.dtype < DT_F32 || t.dtype > DT_F16) return set_error(STT_E_INVALID_ARG, "%s: dtype %d unknown", what, t.dtype);
    if (!t.d_data) return set_error(STT_E_INVALID_ARG, "%s: NULL data", what);
    const int64_t eb = elem_bytes(t.dtype);
    if ((reinterpret_cast<uintptr_t>(t.d_data) | (uint64_t)(t.seq_stride * eb) | (uint64_t)(t.token_stride * eb) |
         (uint64_t)(t.head_stride * eb)) % 16 != 0)
        return set_error(STT_E_INVALID_ARG, "%s must start at, and have strides of, multiples of 16 bytes", what);
    return STT_OK;
}

// A tensor that is written: no two of its rows [n][tokens][heads] of `dim` elements may share memory.  Each
// dimension, from the least stride up, has to step over what the ones before it span.
int check_written(const char* what, const stt_kv8_tensor& t, const stt_kv8_batch& b, int heads, int dim) {
    struct Step {
        __int128 stride;
        int size;
    } d[3] = {{t.seq_stride, b.n}, {t.token_stride, b.n_tokens}, {t.head_stride, heads}};
    for (Step& x : d) x.stride = x.size == 1 ? 0 : x.stride < 0 ? -x.stride : x.stride;
    std::sort(d, d + 3, [](const Step& x, const Step& y) { return x.stride < y.stride; });
    __int128 span = dim;
    for (const Step& x : d) {
        if (x.size == 1) continue;
        if (x.stride < span) return set_error(STT_E_INVALID_ARG, "rows of %s lie on one another", what);
        span += x.stride * (x.size - 1);
    }
    return STT_OK;
}

// A batch's host-side checks; *some is false for one without rows or tokens, which is nothing to do.
int check_batch(const stt_kv8_cache* h, const stt_kv8_batch* b, bool* some) {
    if (!h || !b || b->n < 0 || b->n_tokens < 0) return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (b->n_tokens > INT_MAX - 1024) return set_error(STT_E_INVALID_ARG, "%d tokens are too many for one call", b->n_tokens);
    *some = b->n > 0 && b->n_tokens > 0;
    if (*some && !b->d_pos) return set_error(STT_E_INVALID_ARG, "NULL positions");
    if (!b->d_seqs && b->n > h->c.n_seqs)
        return set_error(STT_E_INVALID_ARG, "%d rows for the %d sequences of the cache", b->n, h->c.n_seqs);
    return STT_OK;
}
Kv8Batch device_batch(const stt_kv8_batch& b) { return Kv8Batch{b.d_seqs, b.d_pos, b.d_count, b.n, b.n_tokens}; }

// K and V of an append or a read.
int check_kv(const stt_kv8_tensor* k, const stt_kv8_tensor* v) {
    if (!k || !v) return set_error(STT_E_INVALID_ARG, "NULL argument");
    TRY(check_tensor("K", *k));
    TRY(check_tensor("V", *v));
    if (k->dtype != v->dtype) return set_error(STT_E_INVALID_ARG, "K has dtype %d, V %d", k->dtype, v->dtype);
    return STT_OK;
}

}  // namespace

int stt::beam_device(const stt_beam* beam) { return beam->device; }
bool stt::beam_fits(const stt_beam* h, int batch, int beams, int vocab) {
    return batch <= h->max_batch && beams <= h->max_beams && vocab <= h->max_vocab;
}

extern "C" int stt_kv8_cache_bytes(int n_seqs, int n_kv_heads, int head_dim, int capacity, size_t* out) {
    clear_error();
    size_t codes, exps;
    if (!out) return set_error(STT_E_INVALID_ARG, "NULL argument");
    if (!kv8_sizes(n_seqs, n_kv_heads, head_dim, capacity, &codes, &exps))
        return set_error(STT_E_INVALID_ARG, "no 8-bit cache of %d sequences, %d heads, head_dim %d (64 or 128), capacity %d (a multiple of %d)",
                         n_seqs, n_kv_heads, head_dim, capacity, kKv8Block);
    *out = 2 * (codes + exps);
    return STT_OK;
}

extern "C" int stt_kv8_cache_create(int device, int n_seqs, int n_kv_heads, int head_dim, int capacity, void* d_memory,
                                    stt_kv8_cache** out) {
    clear_error();
    if (!out) return set_error(STT_E_INVALID_ARG, "NULL argument");
    *out = nullptr;
    size_t bytes = 0, codes = 0, exps = 0;
    TRY(stt_kv8_cache_bytes(n_seqs, n_kv_heads, head_dim, capacity, &bytes));
    kv8_sizes(n_seqs, n_kv_heads, head_dim, capacity, &codes, &exps);
    if (reinterpret_cast<uintptr_t>(d_memory) % 16 != 0)
        return set_error(STT_E_INVALID_ARG, "the cache's memory must be 16-byte aligned");
    DeviceScope ds(device);
    if (!ds.ok) {
        (void)cudaGetLastError();
        return set_error(STT_E_INVALID_ARG, "cannot select device %d", device);
    }
    stt_kv8_cache* h = new (std::nothrow) stt_kv8_cache;
    if (!h) return set_error(STT_E_OOM, "out of host memory");
    h->device = device;
    struct Release {
        stt_kv8_cache*& h;
        ~Release() {
            if (h) stt_kv8_cache_destroy(h);
        }
    } release{h};
    int num_sms = 0;
    CUDA_TRY(cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, device));
    CUDA_TRY(kv8_configure(num_sms, &h->machine));
    if (d_memory) {
        h->memory = d_memory;
    } else {
        ALLOC_TRY(dev_alloc(&h->memory, bytes));
        h->owned = true;
        CUDA_TRY(cudaMemset(h->memory, 0, bytes));
    }
    const size_t tickets = kKv8MaxPartials * sizeof(uint32_t);
    ALLOC_TRY(dev_alloc(&h->scratch, 256 + tickets + kv8_partial_bytes(head_dim)));
    CUDA_TRY(cudaMemset(h->scratch, 0, 256 + tickets));
    CUDA_TRY(cudaDeviceSynchronize());
    uint8_t* s = static_cast<uint8_t*>(h->scratch);
    h->tickets = reinterpret_cast<uint32_t*>(s + 256);
    h->part = reinterpret_cast<float*>(s + 256 + tickets);
    int8_t* m = static_cast<int8_t*>(h->memory);
    h->c = Kv8Dev{m, m + codes, m + 2 * codes, m + 2 * codes + exps, n_seqs, n_kv_heads, head_dim, capacity,
                  reinterpret_cast<int32_t*>(s)};
    *out = h;
    h = nullptr;
    return STT_OK;
}

extern "C" int stt_kv8_cache_destroy(stt_kv8_cache* h) {
    if (!h) return STT_OK;
    {
        DeviceScope ds(h->device);
        if (h->scratch) cudaFree(h->scratch);
        if (h->owned && h->memory) cudaFree(h->memory);
    }
    delete h;
    return STT_OK;
}

extern "C" int stt_kv8_cache_get_info(const stt_kv8_cache* h, stt_kv8_cache_info* o) {
    clear_error();
    if (!h || !o) return set_error(STT_E_INVALID_ARG, "NULL argument");
    *o = stt_kv8_cache_info{h->device, h->c.n_seqs, h->c.heads, h->c.dim, h->c.cap, kKv8Block,
                            h->c.kc, h->c.vc, h->c.ke, h->c.ve};
    return STT_OK;
}

extern "C" int stt_kv8_cache_status(stt_kv8_cache* h) {
    clear_error();
    if (!h) return set_error(STT_E_INVALID_ARG, "NULL argument");
    DeviceScope ds(h->device);
    CUDA_TRY(cudaDeviceSynchronize());
    int32_t code = 0;
    CUDA_TRY(cudaMemcpy(&code, h->c.err, sizeof code, cudaMemcpyDeviceToHost));
    if (code == 0) return STT_OK;
    CUDA_TRY(cudaMemset(h->c.err, 0, sizeof code));
    if (code == STT_E_INVALID_ARG)
        return set_error(code, "a call on this cache had a sequence, position or count out of range, or a sequence "
                               "twice in one append: that row was skipped, or its blocks are undefined");
    return set_error(STT_E_DEVICE_FLAG, "an infinity or NaN was appended to this cache and stored as a finite value, or a wait in "
                                        "an attention kernel ran out");
}

extern "C" int stt_kv8_append_device(stt_kv8_cache* h, const stt_kv8_batch* b, const stt_kv8_tensor* k,
                                     const stt_kv8_tensor* v, void* cuda_stream) {
    clear_error();
    bool some;
    TRY(check_batch(h, b, &some));
    if (!some) return STT_OK;
    TRY(check_kv(k, v));
    if (!b->d_count && b->n_tokens > h->c.cap)  // (counts are the device's to check)
        return set_error(STT_E_INVALID_ARG, "%d tokens in one call exceed the capacity %d", b->n_tokens, h->c.cap);
    if ((int64_t)b->n * (b->n_tokens / kKv8Block + 2) > INT_MAX / (h->c.heads + 8))
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", b->n, b->n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_append(h->c, device_batch(*b), k->d_data, v->d_data, k->dtype, strides(*k), strides(*v),
                               static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_kv8_read_device(const stt_kv8_cache* h, const stt_kv8_batch* b, const stt_kv8_tensor* k,
                                   const stt_kv8_tensor* v, void* cuda_stream) {
    clear_error();
    bool some;
    TRY(check_batch(h, b, &some));
    if (!some) return STT_OK;
    TRY(check_kv(k, v));
    TRY(check_written("K", *k, *b, h->c.heads, h->c.dim));
    TRY(check_written("V", *v, *b, h->c.heads, h->c.dim));
    if (k->d_data == v->d_data) return set_error(STT_E_INVALID_ARG, "K and V are one memory");
    if ((int64_t)b->n * (b->n_tokens / 8 + 1) > INT_MAX / (h->c.heads / 8 + 1))
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", b->n, b->n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_read(h->c, device_batch(*b), k->d_data, v->d_data, k->dtype, strides(*k), strides(*v),
                             static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_kv8_attention_device(stt_kv8_cache* h, const stt_kv8_batch* b, const stt_kv8_tensor* q, int n_heads,
                                        const int32_t* d_start, int window, float scale, const stt_kv8_tensor* out,
                                        void* cuda_stream) {
    clear_error();
    bool some;
    TRY(check_batch(h, b, &some));
    if (window < 0 || !std::isfinite(scale)) return set_error(STT_E_INVALID_ARG, "window %d, scale %g", window, scale);
    if (n_heads <= 0 || n_heads % h->c.heads != 0)
        return set_error(STT_E_INVALID_ARG, "%d query heads over %d K/V heads", n_heads, h->c.heads);
    if (!some) return STT_OK;
    if (!q || !out) return set_error(STT_E_INVALID_ARG, "NULL argument");
    TRY(check_tensor("the queries", *q));
    TRY(check_tensor("the output", *out));
    TRY(check_written("the output", *out, *b, n_heads, h->c.dim));
    Kv8Attention a{};
    a.q = q->d_data;
    a.out = out->d_data;
    a.qs = strides(*q);
    a.os = strides(*out);
    a.q_dtype = q->dtype;
    a.out_dtype = out->dtype;
    a.group = n_heads / h->c.heads;
    a.window = window;
    a.start = d_start;
    a.scale = scale;
    a.part = h->part;
    a.tickets = h->tickets;
    const int64_t rows = (int64_t)b->n_tokens * a.group;
    if (rows > INT_MAX - 256 || (int64_t)b->n * h->c.heads > INT_MAX / (rows / 8 + 1))
        return set_error(STT_E_INVALID_ARG, "%d rows of %d tokens are too many for one call", b->n, b->n_tokens);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_kv8_attention(h->c, device_batch(*b), a, h->machine, static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}

extern "C" int stt_kv8_reorder_device(stt_kv8_cache* h, const int32_t* d_parents, int groups, int beams,
                                      const int32_t* d_held, void* cuda_stream) {
    clear_error();
    if (!h || !d_parents || groups < 0) return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (beams < 1 || beams > kMaxBeams) return set_error(STT_E_INVALID_ARG, "beams %d out of range [1, %d]", beams, kMaxBeams);
    if ((int64_t)groups * beams > h->c.n_seqs)
        return set_error(STT_E_INVALID_ARG, "%d groups of %d beams for the %d sequences of the cache", groups, beams, h->c.n_seqs);
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    // segments: K then V, each head's; the codes in units of a block, then the exponents
    ReorderArgs a{};
    a.segments = 2 * h->c.heads;
    a.inner = h->c.heads;
    a.units = h->c.cap / kKv8Block;
    a.groups = groups;
    a.beams = beams;
    a.parents = d_parents;
    a.held = d_held;
    a.per_unit = kKv8Block;
    for (const bool codes : {true, false}) {
        a.states = reinterpret_cast<uint8_t*>(codes ? h->c.kc : h->c.ke);
        a.unit_bytes = codes ? kKv8Block * h->c.dim : 1;
        a.segment_stride = a.units * a.unit_bytes;
        a.row_stride = a.segment_stride * h->c.heads;
        a.outer_stride = a.row_stride * h->c.n_seqs;
        CUDA_TRY(launch_reorder(a, static_cast<cudaStream_t>(cuda_stream)));
    }
    return STT_OK;
}

// ------------------------------------------------------------------------------------ beam search

extern "C" int stt_beam_create(int device, int max_batch, int max_beams, int max_vocab, stt_beam** out) {
    clear_error();
    if (!out) return set_error(STT_E_INVALID_ARG, "NULL argument");
    *out = nullptr;
    if (max_batch <= 0 || max_beams <= 0 || max_beams > kMaxBeams || max_vocab <= 0)
        return set_error(STT_E_INVALID_ARG, "no selection of %d utterances, %d beams (1..%d), %d tokens", max_batch, max_beams,
                         kMaxBeams, max_vocab);
    if ((int64_t)max_beams * max_vocab > INT_MAX - 4 * beam_tile(DT_BF16) ||
        (int64_t)max_batch * max_beams * beam_max_chunks(max_vocab, DT_F32) > INT_MAX)
        return set_error(STT_E_INVALID_ARG, "%d utterances of %d beams over %d tokens are too many", max_batch, max_beams, max_vocab);
    DeviceScope ds(device);
    if (!ds.ok) {
        (void)cudaGetLastError();
        return set_error(STT_E_INVALID_ARG, "cannot select device %d", device);
    }
    stt_beam* h = new (std::nothrow) stt_beam;
    if (!h) return set_error(STT_E_OOM, "out of host memory");
    h->device = device;
    struct Release {
        stt_beam*& h;
        ~Release() {
            if (h) stt_beam_destroy(h);
        }
    } release{h};
    CUDA_TRY(cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device));
    h->max_batch = max_batch;
    h->max_beams = max_beams;
    h->max_vocab = max_vocab;
    // a call has a CTA for each row, or as many as are resident
    const int64_t rows = (int64_t)max_batch * max_beams;
    const size_t parts = (size_t)std::max(rows, std::min<int64_t>(rows * beam_max_chunks(max_vocab, DT_F32), beam_ctas(DT_F32) * h->num_sms));
    size_t off = 256;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off = (off + bytes + 255) / 256 * 256;
        return o;
    };
    const size_t o_tickets = take((size_t)max_batch * 4), zeroed = off;
    const size_t o_max = take(parts * 4), o_sum = take(parts * 8), o_keys = take(parts * max_beams * 8);
    ALLOC_TRY(dev_alloc(&h->scratch, off));
    CUDA_TRY(cudaMemset(h->scratch, 0, zeroed));
    CUDA_TRY(cudaDeviceSynchronize());
    uint8_t* s = static_cast<uint8_t*>(h->scratch);
    h->err = reinterpret_cast<int32_t*>(s);
    h->ws.tickets = reinterpret_cast<uint32_t*>(s + o_tickets);
    h->ws.part_max = reinterpret_cast<float*>(s + o_max);
    h->ws.part_sum = reinterpret_cast<double*>(s + o_sum);
    h->ws.part_keys = reinterpret_cast<uint64_t*>(s + o_keys);
    h->ws.key_stride = max_beams;
    h->ws.err = h->err;
    *out = h;
    h = nullptr;
    return STT_OK;
}

extern "C" int stt_beam_destroy(stt_beam* h) {
    if (!h) return STT_OK;
    {
        DeviceScope ds(h->device);
        if (h->scratch) cudaFree(h->scratch);
    }
    delete h;
    return STT_OK;
}

extern "C" int stt_beam_status(stt_beam* h) {
    clear_error();
    if (!h) return set_error(STT_E_INVALID_ARG, "NULL argument");
    DeviceScope ds(h->device);
    CUDA_TRY(cudaDeviceSynchronize());
    int32_t code = 0;
    CUDA_TRY(cudaMemcpy(&code, h->err, sizeof code, cudaMemcpyDeviceToHost));
    if (code == 0) return STT_OK;
    CUDA_TRY(cudaMemset(h->err, 0, sizeof code));
    return set_error(STT_E_DEVICE_FLAG, "a beam had a NaN or +inf logit or score (its candidates were taken as -inf), or a wait for "
                                        "logits ran out");
}

extern "C" int stt_beam_select_device(stt_beam* h, const stt_beam_step* s, void* cuda_stream) {
    clear_error();
    return beam_select(h, s, nullptr, static_cast<cudaStream_t>(cuda_stream));
}

int stt::beam_select(stt_beam* h, const stt_beam_step* s, int32_t* err, cudaStream_t st) {
    if (!h || !s || s->batch < 0) return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (s->batch > 0 && (!s->d_logits || !s->d_scores || !s->d_next_scores || !s->d_parents || !s->d_tokens))
        return set_error(STT_E_INVALID_ARG, "NULL array");
    if (s->dtype < DT_F32 || s->dtype > DT_F16) return set_error(STT_E_INVALID_ARG, "dtype %d unknown", s->dtype);
    if (s->beams < 1 || s->vocab < 1 || !beam_fits(h, s->batch, s->beams, s->vocab))
        return set_error(STT_E_INVALID_ARG, "%d utterances, %d beams, %d tokens: the selector was made for %d, %d, %d", s->batch,
                         s->beams, s->vocab, h->max_batch, h->max_beams, h->max_vocab);
    if (s->row_stride < s->vocab)
        return set_error(STT_E_INVALID_ARG, "row stride %lld < vocab %d", (long long)s->row_stride, s->vocab);
    if (s->eos < -1 || s->eos >= s->vocab) return set_error(STT_E_INVALID_ARG, "end token %d outside the %d tokens", s->eos, s->vocab);
    if (s->d_done && s->eos < 0) return set_error(STT_E_INVALID_ARG, "beams that ended need an end token");
    if (reinterpret_cast<uintptr_t>(s->d_logits) % elem_bytes(s->dtype) != 0)
        return set_error(STT_E_INVALID_ARG, "the logits must be aligned to their type");
    if (s->batch == 0) return STT_OK;
    BeamArgs a = h->ws;
    a.logits = s->d_logits;
    a.row_stride = s->row_stride;
    a.batch = s->batch;
    a.beams = s->beams;
    a.vocab = s->vocab;
    // as many CTAs as are resident; a CTA takes whole tiles, and the last one joins a list per thread at most
    // (twice as many lists, each of half the tiles: 8 beams of 128,000 tokens 17 us, where this takes 11.5 us)
    const int tiles = beam_tiles(s->vocab, s->dtype), rows = s->batch * s->beams;
    const int want = std::max(1, std::min({beam_max_chunks(s->vocab, s->dtype), beam_ctas(s->dtype) * h->num_sms / rows,
                                           kBeamThreads / s->beams}));
    a.tiles_per_chunk = (tiles + want - 1) / want;
    a.chunks = (tiles + a.tiles_per_chunk - 1) / a.tiles_per_chunk;
    a.scores = s->d_scores;
    a.done = s->d_done;
    a.eos = s->eos;
    a.next_scores = s->d_next_scores;
    a.parents = s->d_parents;
    a.tokens = s->d_tokens;
    a.next_done = s->d_next_done;
    if (err) a.err = err;
    DeviceScope ds(h->device);
    if (!ds.ok) return set_error(STT_E_CUDA, "cudaSetDevice(%d) failed", h->device);
    CUDA_TRY(launch_beam_select(a, s->dtype, st));
    return STT_OK;
}

extern "C" int stt_beam_reorder_device(int device, const stt_beam_states* s, void* cuda_stream) {
    clear_error();
    if (!s || !s->d_states || !s->d_parents || s->segments < 0 || s->units < 0 || s->unit_bytes <= 0 || s->groups < 0)
        return set_error(STT_E_INVALID_ARG, "bad arguments");
    if (s->beams < 1 || s->beams > kMaxBeams)
        return set_error(STT_E_INVALID_ARG, "beams %d out of range [1, %d]", s->beams, kMaxBeams);
    const __int128 segment = (__int128)s->units * s->unit_bytes;
    const int64_t rows = (int64_t)s->groups * s->beams;
    if (segment > (__int128)1 << 38)
        return set_error(STT_E_INVALID_ARG, "segments of %lld x %lld bytes are too large", (long long)s->units, (long long)s->unit_bytes);
    // rows and segments must not overlap: a position belongs to one of them
    if ((s->segments > 1 && s->segment_stride < segment) || (rows > 1 && s->row_stride < 0))
        return set_error(STT_E_INVALID_ARG, "segments overlap");
    const __int128 row = s->segments == 0 ? 0 : (__int128)(s->segments - 1) * s->segment_stride + segment;
    if (rows > 1 && s->row_stride < row &&
        !(s->row_stride >= segment && s->segment_stride >= (__int128)s->row_stride * (rows - 1) + segment))
        return set_error(STT_E_INVALID_ARG, "rows overlap");
    DeviceScope ds(device);
    if (!ds.ok) {
        (void)cudaGetLastError();
        return set_error(STT_E_INVALID_ARG, "cannot select device %d", device);
    }
    ReorderArgs a{};
    a.states = static_cast<uint8_t*>(s->d_states);
    a.row_stride = s->row_stride;
    a.segment_stride = s->segment_stride;
    a.segments = s->segments;
    a.inner = std::max(1, s->segments);
    a.units = s->units;
    a.unit_bytes = s->unit_bytes;
    a.per_unit = 1;
    a.groups = s->groups;
    a.beams = s->beams;
    a.parents = s->d_parents;
    a.held = s->d_held;
    CUDA_TRY(launch_reorder(a, static_cast<cudaStream_t>(cuda_stream)));
    return STT_OK;
}
